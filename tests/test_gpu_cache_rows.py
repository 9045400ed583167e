"""Rows into the pages of a cache and back, on an MI355X, against the definition: a copy bit for bit, or the codes that
are nearest in exact arithmetic."""
import numpy as np
import pytest

import turboembed_amd as T

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from paged import TYPES, Cache, ints, starts_of, stream  # noqa: E402

BITS = {1: torch.uint8, 2: torch.int16, 4: torch.int32}


def _bits(x):
    return x.contiguous().view(BITS[x.element_size()])


def _same(a, b):
    return torch.equal(_bits(a), _bits(b))


def _new(seed, rows, kv, d, t):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(sum(rows), 2, kv, d, generator=g) * torch.exp(2 * torch.randn(sum(rows), 1, 1, 1, generator=g))
    both = x.to(TYPES[t]).cuda()
    return both[:, 0], both[:, 1]


def _codes(x):
    """The codes and scales of rows by their definition, 64 bits wide (128 where the sides of a border are compared)."""
    x = x.double().cpu().numpy()
    top = np.abs(x).max(-1)
    fine = np.isfinite(x).all(-1)
    safe = np.where(fine & (top > 0), top, 1.0).astype(np.longdouble)[..., None]
    with np.errstate(invalid="ignore"):
        codes = np.rint(127 * np.where(fine[..., None], x, 0.0).astype(np.longdouble) / safe)
    scales = np.where(fine, (top / 127).astype(np.float32), np.float32("nan"))
    return codes.astype(np.int8), scales


def _written(context, cache, k, v, slots):
    before = [x.clone() for x in cache.states + cache.scales if x is not None]
    context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
    kept = torch.ones(cache.slots, dtype=torch.bool, device="cuda")
    kept[slots] = False
    now = [x for x in cache.states + cache.scales if x is not None]
    assert all(_same(a[kept], b[kept]) for a, b in zip(before, now))
    for i, x in enumerate((k, v)):
        if cache.held == "i8":
            codes, scales = _codes(x)
            assert np.array_equal(cache.states[i][slots].cpu().numpy(), codes)
            assert np.array_equal(cache.scales[i][slots].cpu().numpy(), scales, equal_nan=True)
        else:
            assert _same(cache.states[i][slots], x)


def _read(context, cache, out_type):
    k, v = (torch.full((sum(cache.rows), cache.kv, cache.d), 7.0, dtype=out_type, device="cuda") for _ in "kv")
    context.cache_read(cache.operand(T), *cache.arrays(), k, v, stream=stream())
    return k, v


SETS = [((1,), (1,)), ((1, 1, 1), (5, 64, 200)), ((3, 0, 9), (3, 17, 90)), ((70,), (300,)), ((1,) * 130, tuple(range(1, 131))),
        ((200, 1, 37), (200, 1, 40))]


@pytest.mark.parametrize("rows, lengths", SETS, ids=lambda x: "-".join(map(str, x[:4])))
@pytest.mark.parametrize("kv, d, page", [(1, 64, 16), (3, 80, 24), (8, 128, 64), (2, 32, 1), (5, 7, 100)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_rows_there_and_back(context, rows, lengths, kv, d, page, t, held):
    cache = Cache(1, rows, lengths, kv, d, t, held, page)
    k, v = _new(2, rows, kv, d, t)
    slots = cache.new_slots()
    _written(context, cache, k, v, slots)
    for out_type in [TYPES[t]] if held == "same" else TYPES.values():
        for i, got in enumerate(_read(context, cache, out_type)):
            if held == "same":
                assert _same(got, (k, v)[i])
                continue
            # (8-bit codes by 24-bit scales: exact in 64 bits, so rounded once here too.)
            exact = cache.states[i][slots].double() * cache.scales[i][slots].double()[..., None]
            want = torch.from_numpy(_once(exact.cpu().numpy(), out_type)).cuda()
            assert torch.equal(got.double(), want)


@pytest.mark.parametrize("kv, d", [(13, 32), (13, 20), (7, 64), (9, 43), (5, 128), (5, 101)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_long_calls(context, kv, d, t, held):
    """Rows enough for every kernel of long calls, a number that no workgroup divides, some of them nobody's and some
    without a place."""
    rows = (3001, 1, 0, 2500, 77)
    cache = Cache(1, rows, (3300, 1, 5, 2500, 100), kv, d, t, held, 16)
    k, v = _new(2, (sum(rows) + 11,), kv, d, t)
    slots = cache.new_slots()
    cache.starts += 6
    cache.pages[3, 40:50] = -1                                # tokens 640 to 799 of sequence 3
    there = torch.ones(sum(rows), dtype=torch.bool, device="cuda")
    there[3002 + 640:3002 + 800] = False
    context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
    for out_type in [TYPES[t]] if held == "same" else TYPES.values():
        got = [torch.full((len(k), kv, d), 7.0, dtype=out_type, device="cuda") for _ in "kv"]
        context.cache_read(cache.operand(T), *cache.arrays(), *got, stream=stream())
        for i, (g, x) in enumerate(zip(got, (k, v))):
            assert (g[:6] == 7).all() and (g[-5:] == 7).all()
            mine, x = g[6:-5], x[6:-5]
            assert (mine[~there] == 0).all()
            if held == "same":
                assert _same(mine[there], x[there]) and _same(cache.states[i][slots[there]], x[there])
                continue
            codes, scales = _codes(x[there])
            assert np.array_equal(cache.states[i][slots[there]].cpu().numpy(), codes)
            assert np.array_equal(cache.scales[i][slots[there]].cpu().numpy(), scales)
            want = _once(codes.astype(np.float64) * scales.astype(np.float64)[..., None], out_type)
            assert np.array_equal(mine[there].double().cpu().numpy(), want)


def _once(x, t):
    """64-bit numbers to the nearest of type t, ties to even, as 64-bit numbers."""
    f = torch.finfo(t)
    m, e = np.frexp(np.abs(x))
    low = int(np.round(np.log2(f.tiny)))
    step = np.exp2(np.maximum(e - 1, low) + np.log2(f.eps))
    return np.copysign(np.rint(np.abs(x) / step) * step, x)


@pytest.mark.parametrize("d", [1, 2, 3, 8, 9, 31, 33, 40, 63, 65, 100, 127])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_every_kind_of_width(context, d, held):
    for t in TYPES:
        cache = Cache(d, (5, 2), (20, 2), 3, d, t, held, 8)
        _written(context, cache, *_new(d, (5, 2), 3, d, t), cache.new_slots())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_codes_of_rows_of_every_kind(context, t):
    d = 64
    cache = Cache(3, (64,), (64,), 2, d, t, "i8", 16)
    k, v = (x.clone() for x in _new(4, (64,), 2, d, t))
    top = torch.finfo(TYPES[t]).max
    k[0] = 0
    k[1, 0, 5], k[2, 1, 63], k[3, 0, 0] = float("nan"), float("inf"), -float("inf")
    k[4] = torch.linspace(-top, top, d, dtype=torch.float64).to(TYPES[t])
    k[5] = torch.finfo(TYPES[t]).tiny * torch.randn(d, device="cuda")
    k[6] = torch.finfo(TYPES[t]).smallest_normal * torch.finfo(TYPES[t]).eps * torch.arange(d, device="cuda")
    # Quotients next to and on the borders of two codes.
    k[7] = ((torch.arange(d) * 4 - 127) / 2).to(TYPES[t])
    k[7, :, 0] = 127
    for i in range(8, 64):
        k[i] = (torch.arange(d) + 0.5).to(TYPES[t]) * (1 + i / 64)
        k[i, :, 1] = 127 * (1 + i / 64)
    _written(context, cache, k, v, cache.new_slots())


def test_tokens_without_a_place_are_not_written_and_read_as_zeros(context):
    page, kv, d = 4, 2, 32
    for held in ("same", "i8"):
        cache = Cache(5, (6, 3, 5, 2), (9, 7, 10, 2), kv, d, "f16", held, page)
        k, v = _new(6, (6, 3, 5, 2), kv, d, "f16")
        whole = cache.new_slots().split([6, 3, 5, 2])
        # Sequence 0 has fewer states than new tokens: its first two are none. 1: a page that the cache does not have.
        # 2: a length past its table. 3: no states at all.
        cache.lengths.copy_(ints([4, 7, 11, -3]))
        count = cache.slots // page
        cache.pages[1, 1] = count
        cache.pages[2, 2] = -2147483648
        first = cache.at(0, 0, 4)
        third = cache.at(2, 6, 8)
        slots = torch.cat([first, third])
        rows = torch.tensor([2, 3, 4, 5, 9, 10], device="cuda")
        kk, vv = k[rows], v[rows]
        before = [x.clone() for x in cache.states + cache.scales if x is not None]
        context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
        kept = torch.ones(cache.slots, dtype=torch.bool, device="cuda")
        kept[slots] = False
        assert all(_same(a[kept], b[kept])
                   for a, b in zip(before, [x for x in cache.states + cache.scales if x is not None]))
        cache.rows = (6, 3, 5, 2)
        gk, gv = _read(context, cache, torch.float16)
        nothing = torch.ones(16, dtype=torch.bool, device="cuda")
        nothing[rows] = False
        for got, x in ((gk, kk), (gv, vv)):
            assert (got[nothing] == 0).all()
            if held == "same":
                assert _same(got[rows], x)
            else:
                assert ((got[rows].float() - x.float()).abs() <= x.float().abs().amax(-1, keepdim=True) * 0.0045).all()
        assert len(whole) == 4


def test_rows_of_no_sequence_are_left(context):
    kv, d = 2, 16
    cache = Cache(7, (3, 4), (8, 4), kv, d, "bf16", "same", 4)
    k, v = _new(8, (12,), kv, d, "bf16")
    # Rows 0 and 1, and 9 to 11, are nobody's.
    cache.starts.copy_(ints([2, 5, 9]))
    context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
    assert _same(cache.states[0][cache.new_slots()], k[2:9]) and _same(cache.states[1][cache.new_slots()], v[2:9])
    gk, gv = (torch.full((12, kv, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    context.cache_read(cache.operand(T), *cache.arrays(), gk, gv, stream=stream())
    assert _same(gk[2:9], k[2:9]) and _same(gv[2:9], v[2:9])
    for x in (gk, gv):
        assert (x[:2] == 7).all() and (x[9:] == 7).all()
    # Starts that point outside of the call's rows, and that descend.
    for bad in ([-5, 3, 90], [2147483647, -2147483648, 5], [9, 2, 12]):
        cache.starts.copy_(ints(bad))
        context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
        context.cache_read(cache.operand(T), *cache.arrays(), gk, gv, stream=stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("held", ["same", "i8"])
def test_layouts(context, held):
    rows, lengths, kv, d, page = (5, 40), (50, 40), 3, 40, 8
    for t in TYPES:
        plain = Cache(9, rows, lengths, kv, d, t, held, page)
        k, v = _new(10, rows, kv, d, t)
        _written(context, plain, k, v, plain.new_slots())
        # K and V side by side in a slot; head by head; columns of wider rows that start at any element.
        n = plain.slots
        dtype = plain.states[0].dtype
        side = torch.empty(n, 2, kv, d, dtype=dtype, device="cuda")
        hm = torch.empty(2, kv, n, d, dtype=dtype, device="cuda")
        wide = torch.empty(n, 2 * kv * d + 13, dtype=dtype, device="cuda")
        scales = torch.empty(n, 2 * kv + 1, device="cuda")
        for ck, cv in ((side[:, 0], side[:, 1]), (hm[0].transpose(0, 1), hm[1].transpose(0, 1)),
                       (wide[:, 3:3 + kv * d].unflatten(1, (kv, d)), wide[:, 5 + kv * d:5 + 2 * kv * d].unflatten(1, (kv, d)))):
            cache = Cache(9, rows, lengths, kv, d, t, held, page)
            for x, y in zip((ck, cv), cache.states):
                x.copy_(y)
            cache.states = [ck, cv]
            if held == "i8":
                sk, sv = scales[:, 1:1 + kv], scales[:, 1 + kv:]
                sk.copy_(cache.scales[0]), sv.copy_(cache.scales[1])
                cache.scales = [sk, sv]
            _written(context, cache, k, v, cache.new_slots())
            kk, vv = (torch.empty(sum(rows), 2 * kv * d + 1, dtype=TYPES[t], device="cuda")[:, 1:] for _ in "kv")
            kk, vv = (x[:, :kv * d].unflatten(1, (kv, d)) for x in (kk, vv))
            context.cache_read(cache.operand(T), *cache.arrays(), kk, vv, stream=stream())
            want = _read(context, plain, TYPES[t])
            assert _same(kk, want[0]) and _same(vv, want[1])


def test_slots_past_32_bits(context):
    # 20 pages of 16 slots, 16 MiB from one to the next.
    kv, d, page, step = 1, 64, 16, 1 << 23
    pool = torch.empty(20 * page * step, dtype=torch.float16, device="cuda")
    ck = pool.as_strided((20 * page, kv, d), (step, d, 1))
    cv = pool.as_strided((20 * page, kv, d), (step, d, 1), 128)
    pages = ints([[19, 0, 18]])
    k, v = _new(11, (40,), kv, d, "f16")
    operand = T.StateCache(ck, cv, page)
    context.cache_write(k, v, operand, starts_of([40]), ints([40]), pages, stream=stream())
    at = torch.cat([torch.arange(p * page, p * page + page, device="cuda") for p in (19, 0, 18)])[:40]
    assert _same(ck[at], k) and _same(cv[at], v)
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    context.cache_read(operand, starts_of([40]), ints([40]), pages, gk, gv)      # the context's own stream, waited for
    assert _same(gk, k) and _same(gv, v)


def test_nothing_to_do(context):
    for held in ("same", "i8"):
        cache = Cache(12, (0, 0), (5, 0), 2, 32, "f16", held, 4)
        k = torch.empty(0, 2, 32, dtype=torch.float16, device="cuda")
        context.cache_write(k, k, cache.operand(T), *cache.arrays(), stream=stream())
        context.cache_read(cache.operand(T), *cache.arrays(), k, k.clone(), stream=stream())
    # No sequences; a cache without a page.
    k = torch.full((3, 2, 32), 5.0, dtype=torch.float16, device="cuda")
    none = torch.empty(0, 2, 32, dtype=torch.float16, device="cuda")
    for starts, lengths, pages in (([0], [], (0, 4)), ([0, 2], [2], (1, 0)), ([0, 2], [2], (1, 3))):
        for pool in (none, k.new_zeros(3, 2, 32)):
            table = torch.zeros(pages, dtype=torch.int32, device="cuda")
            args = T.StateCache(pool, pool.clone(), 4), ints(starts), ints(lengths), table
            context.cache_write(k, k, *args, stream=stream())
            out = torch.full_like(k, 3.0), torch.full_like(k, 3.0)
            context.cache_read(*args, *out, stream=stream())
            assert (pool == 0).all()
            for x in out:
                assert (x[:len(lengths) and 2] == 0).all() and (x[len(lengths) and 2:] == 3).all()


@pytest.mark.parametrize("held", ["same", "i8"])
def test_captured_with_arrays_that_change(context, held):
    rows, kv, d, page = (1, 1, 1), 2, 64, 4
    cache = Cache(13, rows, (5, 9, 16), kv, d, "bf16", held, page)
    k, v = _new(14, rows, kv, d, "bf16")
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
        context.cache_read(cache.operand(T), *cache.arrays(), gk, gv, stream=stream())
    for step in range(4):
        nk, nv = _new(20 + step, rows, kv, d, "bf16")
        k.copy_(nk), v.copy_(nv)
        cache.lens = [5 - step, 9 - step, 16 - step]
        cache.lengths.copy_(ints(cache.lens))
        gk.zero_(), gv.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = _read(context, cache, torch.bfloat16)
        assert _same(gk, want[0]) and _same(gv, want[1])
        slots = cache.new_slots()
        if held == "same":
            assert _same(cache.states[0][slots], nk) and _same(cache.states[1][slots], nv)
        else:
            assert np.array_equal(cache.states[1][slots].cpu().numpy(), _codes(nv)[0])


@pytest.mark.parametrize("n", [70, 5000])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_many_empty_sequences_between_the_tokens(context, n, held):
    rows, lengths = [0] * n, [0] * n
    for i, m in ((0, 1), (1, 2), (n // 2, 1), (n // 2 + 17, 3), (n - 4, 90), (n - 2, 1)):
        rows[i], lengths[i] = m, m + 20
    cache = Cache(1, rows, lengths, 3, 64, "bf16", held, 16)
    k, v = _new(2, rows, 3, 64, "bf16")
    slots = cache.new_slots()
    _written(context, cache, k, v, slots)
    for x, y in zip(_read(context, cache, torch.bfloat16), (0, 1)):
        assert torch.equal(x, cache.values(y, slots).to(torch.bfloat16))
