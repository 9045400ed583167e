"""The kernels of a prompt's attention and of attention over a cache, one by one, on an MI355X against 64-bit arithmetic:
what each holds its weights in, at every padded width, with windows, values that are no numbers, strides and replays."""
import pytest

import turboembed_amd as T
from turboembed_amd import operators as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from paged import TYPES, Cache, ints, starts_of, stream  # noqa: E402
from test_self_kernels import BYTES, CHUNKS as WHOLE, CODES, INT8, LOOSE, PROMPT, SAME  # noqa: E402

# A weight's error against itself. F32: none of its own. Rounded once: half a step. As the sum of two numbers: the first is
# less than two steps below the weight, the second what is left, rounded once: half a step of two steps.
ONCE = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TWO = {"f32": 0.0, "f16": 2.0 ** -11 * 2.0 ** -9, "bf16": 2.0 ** -8 * 2.0 ** -6}


def rows_of(seed, n, heads, d, t, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, d, generator=g) * spread).to(TYPES[t]).cuda()


def check(out, q, first, k, v, kept, window=0, scale=None, unit=None):
    """out is the attention of q's rows at positions first .. to the states k and v [n, kv, d] (64 bits).

    A score is a sum of d F32 products times one or two factors, less a maximum: off by at most e = (d + 6) 2^-24 A + 2^-22 S, A
    the largest sum of |q_c k_c| scale and S the largest |score| of the row. A weight is off by a factor of 1 +- (2 e + 2^-21)
    against its row's sum and by `kept` of itself, and, in F16, by half the smallest number, 2^-25 of the row's largest. Of int8
    values the scale is part of it, against a unit of at most 4 times the largest that the row sees: `unit` [m, 1], for each
    of n codes. Sums of n products are off by n 2^-24 each, and the output is rounded once."""
    m, heads, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    if m == 0:
        return
    scale = d ** -0.5 if scale is None else scale
    half, tiny = torch.finfo(out.dtype).eps / 2, torch.finfo(out.dtype).tiny
    at, p = first + torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    live = p[None] <= at[:, None]
    if window:
        live &= p[None] > at[:, None] - window
    seen = live.any(0)[:, None, None]
    none = ~live.any(1)
    assert (out[none] == 0).all()
    if none.all():
        return
    # (States that no row sees may hold anything.)
    k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
    share, step = heads // kv, max(1, (1 << 24) // (m * n * (heads // kv)))
    for h0 in range(0, kv, step):                 # (some key heads at a time)
        h1 = min(kv, h0 + step)
        one = lambda x: x[:, h0 * share:h1 * share].double().unflatten(1, (h1 - h0, share)).permute(1, 2, 0, 3)  # noqa: E731
        qs, o = one(q).flatten(1, 2).contiguous(), one(out)
        kk, vv = k[:, h0:h1].permute(1, 2, 0).contiguous(), v[:, h0:h1].transpose(0, 1).contiguous()
        s = torch.matmul(qs, kk).mul_(scale).unflatten(1, (share, m)).masked_fill_(~live, -float("inf"))
        pr = torch.softmax(s, -1).nan_to_num_(0.0)
        want = torch.matmul(pr.flatten(1, 2), vv).unflatten(1, (share, m))
        a = torch.matmul(qs.abs(), kk.abs()).unflatten(1, (share, m)).masked_fill_(~live, 0).amax(-1, keepdim=True)
        big = s.abs().masked_fill_(~live, 0).amax(-1, keepdim=True)
        off = 2 * ((d + 6) * 2.0 ** -24 * a * abs(scale) + 2.0 ** -22 * big) + 2.0 ** -21 + n * 2.0 ** -23 + kept
        weight = torch.matmul((pr * off).flatten(1, 2), vv.abs()).unflatten(1, (share, m))
        if out.dtype == torch.float16:
            each = vv.abs().sum(1)[:, None, None] if unit is None else 127.0 * n * unit
            weight = weight + 2.0 ** -25 * pr.amax(-1, keepdim=True) * each
        tol = weight * 1.01 + want.abs().clamp_min(tiny) * half * 1.01
        o, want, tol = o[:, :, ~none], want[:, :, ~none], tol[:, :, ~none]
        assert torch.isfinite(o).all()
        worst = ((o - want).abs() / tol).max().item()
        assert worst <= 1, (m, n, h0, worst)


def check_prompt(out, q, k, v, rows, kept, window=0, scale=None):
    at = 0
    for m in rows:
        check(out[at:at + m], q[at:at + m], 0, k[at:at + m].double(), v[at:at + m].double(), kept, window, scale)
        at += m


def prompt(context, q, k, v, rows, kept, window=0, scale=None, out=None):
    out = torch.full_like(q, 3.0) if out is None else out
    context.prompt_attention(q, k, v, starts_of(rows), out, window=window, scale=scale, stream=stream())
    check_prompt(out, q, k, v, rows, kept, window, scale)
    return out


@pytest.mark.parametrize("rows", [(1,), (23,), (33,), (5, 0, 90), (300, 7)], ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads, kv, d", [(12, 12, 64), (4, 1, 32), (3, 3, 80), (8, 2, 128)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_prompts_of_few_rows_carry_weights_as_two_numbers(context, rows, heads, kv, d, t):
    n = sum(rows)
    q, k, v = rows_of(n, n, heads, d, t), rows_of(n + 1, n, kv, d, t), rows_of(n + 2, n, kv, d, t)
    for window in (0, 40):
        prompt(context, q, k, v, rows, TWO[t], window)


@pytest.mark.parametrize("n", [65, 300, 2048])
@pytest.mark.parametrize("heads, kv, d", [(1, 1, 80), (3, 3, 40), (2, 1, 24), (8, 4, 112)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_padded_heads_of_more_sequences_than_a_wave(context, n, heads, kv, d, t):
    """Columns past the width are cleared in the bytes where such a prompt's blocks are counted: no count may be lost."""
    rows = [1 + 7 * i % 5 for i in range(n)]
    rows[3], rows[n // 2], rows[-1] = 0, 150, 70
    m = sum(rows)
    q, k, v = rows_of(n, m, heads, d, t), rows_of(n + 1, m, kv, d, t), rows_of(n + 2, m, kv, d, t)
    outs = [torch.full_like(q, float("nan")) for _ in range(4)]
    for out in outs:
        context.prompt_attention(q, k, v, starts_of(rows), out, stream=stream())
    same = all(torch.equal(outs[0], out) for out in outs)
    assert same
    ends = torch.tensor(rows).cumsum(0).tolist()
    for i in sorted({0, 1, 2, 3, 4, 63, 64, n // 2 - 1, n // 2, n // 2 + 1, n - 2, n - 1} | set(range(0, n, n // 30))):
        a, b = ends[i] - rows[i], ends[i]
        check(outs[0][a:b], q[a:b], 0, k[a:b].double(), v[a:b].double(), ONCE[t])
    assert torch.isfinite(outs[0]).all()


def attend(context, cache, q, window=0, scale=None, out=None):
    out = torch.full_like(q, 3.0) if out is None else out
    need = context.cache_workspace(len(q), len(cache.rows), q.shape[1], cache.kv, cache.d, cache.dtype)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    context.cache_attention(q, cache.operand(T), *cache.arrays(), out, window=window, scale=scale, workspace=ws, stream=stream())
    return out


# Calls of 16, 32 and 128 rows a block.
CHUNKS = [((1,), (700,)), ((12,), (90,)), ((20,), (90,)), ((40,), (40,)), ((300,), (300,)), ((300,), (1500,))]


@pytest.mark.parametrize("rows, lengths", CHUNKS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("window", [0, 9, 200])
@pytest.mark.parametrize("way", ["up", "down", "first"])
@pytest.mark.parametrize("d", [64, 40])
def test_f16_rows_over_int8_values_of_sizes_that_change(context, rows, lengths, window, way, d):
    """Every row against the largest scale that it sees itself."""
    (m,), (n,) = rows, lengths
    cache = Cache(m, rows, lengths, 2, d, "f16", "i8", 16)
    p, at = torch.arange(n, device="cuda"), cache.at(0, 0, n)
    size = {"up": torch.exp2(p * 12.0 / n - 13), "down": torch.exp2(-p * 12.0 / n - 1),
            "first": torch.where(p == 0, 2.0 ** -30, 0.02)}[way]
    cache.scales[1][at] = size[:, None].expand(n, 2).contiguous()
    q = rows_of(m, m, 4, d, "f16")
    out = attend(context, cache, q, window)
    pos = n - m + torch.arange(m, device="cuda")
    live = (p[None] <= pos[:, None]) & (p[None] > pos[:, None] - (window or n))
    unit = 4 * torch.where(live, size[None], 0.0).amax(1, keepdim=True).double()
    # (Two heads of a key head: more than 32 rows of a sequence are four waves', whose weights are rounded once.)
    kept = ONCE["f16"] if 2 * m > 32 else TWO["f16"]
    check(out, q, n - m, cache.values(0, at), cache.values(1, at), kept, window, unit=unit)


@pytest.mark.parametrize("m, n", [(20, 30), (40, 40), (300, 300)])
def test_a_value_that_is_large_and_weighs_nothing(context, m, n):
    """A finite scale of 2^100 whose weight is 0 leaves the rows that see it finite, and the others' bits as they are."""
    cache = Cache(1, (m,), (n,), 1, 64, "f16", "i8", 16)
    q = rows_of(2, m, 2, 64, "f16")
    q[:, :, 0] = 1.0
    at = n - m // 2
    slot = cache.at(0, at, at + 1)
    cache.scales[1][cache.at(0, 0, 1)] = 0.0
    before = attend(context, cache, q, scale=1.0)
    cache.states[0][slot] = 0
    cache.states[0][slot, 0, 0] = -127
    cache.scales[0][slot] = 4.0                # (a score of -508)
    cache.scales[1][slot] = 2.0 ** 100
    out = attend(context, cache, q, scale=1.0)
    fine = torch.isfinite(out).all()
    assert fine
    same = torch.equal(out[:at - (n - m)], before[:at - (n - m)])
    assert same


def _time(f):
    f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        graph.replay()
        a.record()
        for _ in range(5):
            graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("window, first", [(64, 1.0), (1024, 1.0), (0, 2.0 ** -12)])
def test_f16_rows_over_int8_values_take_bf16_s_time(context, window, first):
    """Windows, and a first value that is small, cost F16 rows no more than others: half as much again at most."""
    took = {}
    rows, lengths = (512,) * 4, (512,) * 4 if first < 1 else (1024, 3000, 5000, 8192)
    for t in ("f16", "bf16"):
        cache = Cache(1, rows, lengths, 8, 64, t, "i8", 32)
        for i in range(4):
            cache.scales[1][cache.at(i, 0, 1)] *= first
        q = rows_of(2, 2048, 8, 64, t)
        ws = torch.empty(context.cache_workspace(2048, 4, 8, 8, 64, TYPES[t]), dtype=torch.uint8, device="cuda")
        operand, arrays, out = cache.operand(T), cache.arrays(), torch.empty_like(q)
        took[t] = _time(lambda: context.cache_attention(q, operand, *arrays, out, window=window, workspace=ws, stream=stream()))
    assert took["f16"] <= 1.5 * took["bf16"], took


def _among(n, live):
    """n sequences of which a few have a token, or more."""
    rows, lengths = [0] * n, [0] * n
    for i, m, s in live:
        rows[i], lengths[i] = m, s
    return rows, lengths


@pytest.mark.parametrize("t, held", [("f32", "same"), ("bf16", "same"), ("f16", "i8")])
@pytest.mark.parametrize("many", [0, 40])
def test_a_few_tokens_among_many_idle_sequences(context, t, held, many):
    rows, lengths = _among(5000, ((0, 1, 400), (1, 1, 30), (64, 1, 90), (700, many, 900), (701, 1, 64), (2900, 1, 3000), (4998, 2, 5)))
    cache = Cache(1, rows, lengths, 2, 64, t, held, 16)
    q = rows_of(2, sum(rows), 4, 64, t)
    out, at = attend(context, cache, q), 0
    for i, (m, s) in enumerate(zip(rows, lengths)):
        if m:
            where = cache.at(i, 0, s)
            unit = 4 * cache.scales[1][where].amax().double() * torch.ones(m, 1, device="cuda") if held == "i8" else None
            check(out[at:at + m], q[at:at + m], s - m, cache.values(0, where), cache.values(1, where), ONCE[t], unit=unit)
            at += m


def test_idle_sequences_between_two_take_no_time_each(context):
    """Two live sequences behind 20,000 idle ones, and one of them before those: four times the time at most."""
    n, took = 20002, []
    for first in (n - 2, 0):
        rows, lengths = _among(n, ((first, 1, 200), (n - 1, 1, 200)))
        cache = Cache(1, rows, lengths, 1, 64, "bf16", "same", 16)
        q, ws = rows_of(2, 2, 4, 64, "bf16"), torch.empty(context.cache_workspace(2, n, 4, 1, 64, torch.bfloat16), dtype=torch.uint8, device="cuda")
        operand, arrays, out = cache.operand(T), cache.arrays(), torch.empty_like(q)
        took.append(_time(lambda: context.cache_attention(q, operand, *arrays, out, workspace=ws, stream=stream())))
    assert took[1] <= 4 * took[0], took


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_keys_and_values_next_to_each_other(context, t, held):
    """Head by head in a slot, in a head, and in a head's plane: written, read back and attended to as apart."""
    rows, lengths, kv, d = (5, 40), (50, 40), 3, 40
    plain = Cache(9, rows, lengths, kv, d, t, held, 8)
    k, v, q = (rows_of(s, 45, h, d, t) for s, h in ((1, kv), (2, kv), (3, 6)))

    def step(cache):
        out = [torch.empty_like(k), torch.empty_like(v)]
        context.cache_write(k, v, cache.operand(T), *cache.arrays(), stream=stream())
        context.cache_read(cache.operand(T), *cache.arrays(), *out, stream=stream())
        return [*out, attend(context, cache, q), *(x[cache.new_slots()].clone() for x in cache.states)]
    n, dtype = plain.slots, plain.states[0].dtype
    before = [x.clone() for x in plain.states]
    want = step(plain)
    for shape, axes in (((n, kv, 2, d), (0, 1, 2)), ((kv, n, 2, d), (1, 0, 2)), ((kv, 2, n, d), (2, 0, 1))):
        both = torch.empty(shape, dtype=dtype, device="cuda").permute(*axes, 3)
        cache = Cache(9, rows, lengths, kv, d, t, held, 8)
        cache.states = [both[:, :, 0], both[:, :, 1]]
        for x, y in zip(cache.states, before):
            x.copy_(y)
        for got, w in zip(step(cache), want):
            same = torch.equal(got, w)
            assert same


# ---- the kernels of long prompts -----------------------------------------------------------

# 70 sequences of 40 to 120 tokens, and a few long ones, of so many key heads that blocks of 128 rows (F32: of 32, a wave
# each) fill the card.
MANY, LONG = (tuple(40 + 80 * i // 69 for i in range(70)), 8), ((300, 900, 65, 128, 513, 0, 700, 641), 16)


def _long(rows, heads, kv, d, t):
    n = sum(rows)
    assert O.self_kernel(n, len(rows), heads, kv, d, TYPES[t]) == ((32, 1, WHOLE) if t == "f32" else (128, 4, WHOLE))
    return rows_of(n, n, heads, d, t), rows_of(n + 1, n, kv, d, t), rows_of(n + 2, n, kv, d, t)


@pytest.mark.parametrize("d", [24, 32, 40, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_long_prompts_of_every_padded_width(context, d, t):
    for (rows, kv), share in ((MANY, 4), (LONG, 2)):
        q, k, v = _long(rows, share * kv, kv, d, t)
        for window in (0, 1, 50, 300):
            prompt(context, q, k, v, rows, ONCE[t], window)


JUNK = (float("nan"), float("inf"), -float("inf"), 1e30)


@pytest.mark.parametrize("rows, kv", [MANY, LONG], ids=["many", "long"])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_long_prompts_do_not_see_later_tokens_whatever_they_hold(context, rows, kv, d, t):
    """One token in each sequence's middle holds no numbers: the rows before it, and those past its window, are the formula's."""
    q, k0, v0 = _long(rows, 2 * kv, kv, d, t)
    for junk, window in zip(JUNK + JUNK, (0, 9, 70, 0, 130, 0, 9, 9)):
        k, v, at = k0.clone(), v0.clone(), 0
        for m in rows:
            if m:
                v[at + m // 2], k[at + m // 2, :, 3] = junk, junk
            at += m
        out = torch.full_like(q, 3.0)
        context.prompt_attention(q, k, v, starts_of(rows), out, window=window, stream=stream())
        at = 0
        for m in rows:
            j = m // 2
            check(out[at:at + j], q[at:at + j], 0, k[at:at + j].double(), v[at:at + j].double(), ONCE[t], window)
            if window and j + window < m:
                a, b = at + j + 1, at + m        # (the states from behind it on)
                past = at + j + window
                check(out[past:b], q[past:b], window - 1, k[a:b].double(), v[a:b].double(), ONCE[t], window)
            at += m


@pytest.mark.parametrize("scale", [0.0, -0.5, 1.0, 1e-30])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_long_prompts_scales(context, scale, t):
    for (rows, kv), d in ((MANY, 64), (LONG, 80)):
        q, k, v = _long(rows, 2 * kv, kv, d, t)
        prompt(context, q, k, v, rows, ONCE[t], scale=scale)


@pytest.mark.parametrize("d", [32, 64, 80, 128])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_long_prompts_layouts(context, d, t):
    """Every layout gives the same bits."""
    rows, kv = MANY
    heads, n = 2 * kv, sum(rows)
    q, k, v = _long(rows, heads, kv, d, t)
    want = prompt(context, q, k, v, rows, ONCE[t], 70)

    def head_major(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    def wider(x, off, by):      # rows of more columns, of which x has some
        y = torch.full((n, x.shape[1] * d + by), 2.0, dtype=x.dtype, device="cuda")[:, off:off + x.shape[1] * d].unflatten(1, (x.shape[1], d))
        y.copy_(x)
        return y
    side = torch.cat([q, k, v], 1).split([heads, kv, kv], 1)
    between = torch.stack([k, v], 2)
    for a, b, c in ((head_major(q), head_major(k), head_major(v)), side, (wider(q, 1, 7), wider(k, 16, 32), wider(v, 8, 8)),
                    (q, between[:, :, 0], between[:, :, 1])):
        for out in (torch.empty_like(q), wider(q, 5, 11), head_major(q).clone()):
            out.fill_(3.0)
            context.prompt_attention(a, b, c, starts_of(rows), out, window=70, stream=stream())
            same = torch.equal(out, want)
            assert same
    # One key head for all, and rows of the call that are nobody's.
    k1, v1 = (x[:, :1].expand(n, kv, d) for x in (k, v))
    prompt(context, q, k1, v1, rows, ONCE[t])
    fewer, out = rows[:-1], torch.full_like(q, 3.0)
    context.prompt_attention(q, k, v, starts_of(fewer), out, window=70, stream=stream())
    same = torch.equal(out[:sum(fewer)], want[:sum(fewer)]) and bool((out[sum(fewer):] == 3).all())
    assert same


@pytest.mark.parametrize("d", [64, 80])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_long_prompts_captured_with_starts_that_change(context, d, t):
    rows, kv = MANY
    q, k, v = _long(rows, 2 * kv, kv, d, t)
    n, starts, out = sum(rows), starts_of(rows), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        context.prompt_attention(q, k, v, starts, out, window=200, stream=stream())
    for again in range(4):
        now = rows[again:] + rows[:again] if again < 3 else (1,) * 69 + (n - 69,)
        starts.copy_(starts_of(now))
        q.copy_(rows_of(50 + again, n, 2 * kv, d, t))
        out.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_prompt(out, q, k, v, now, ONCE[t], 200)
        first = out.clone()
        context.prompt_attention(q, k, v, starts, out, window=200, stream=stream())
        same = torch.equal(first, out)
        assert same


# ---- every kernel of a call over a cache ---------------------------------------------------

def check_cache(cache, q, out, kept, window=0):
    at = 0
    for i, (m, n) in enumerate(zip(cache.rows, cache.lens)):
        where, unit = cache.at(i, 0, n), None
        if cache.held == "i8":
            p, pos = torch.arange(n, device="cuda"), n - m + torch.arange(m, device="cuda")
            live = (p[None] <= pos[:, None]) & (p[None] > pos[:, None] - (window or n))
            unit = 4 * torch.where(live, cache.scales[1][where].amax(1)[None].double(), 0.0).amax(1, keepdim=True)
        check(out[at:at + m], q[at:at + m], n - m, cache.values(0, where), cache.values(1, where), kept, window, unit=unit)
        at += m


OVER = [(t, states, rows) for t in ("f32", "f16", "bf16") for states in (SAME, INT8) for rows in (16, 32, 128) if (t, rows) != ("f32", 16)]


@pytest.mark.parametrize("d", [24, 32, 33, 48, 64, 80, 91, 96, 112, 127, 128])
@pytest.mark.parametrize("t, states, rows", OVER)
def test_every_kernel_of_a_call_over_a_cache(context, t, states, rows, d):
    """One token, a few and many, two heads to a key head; pages that a tile divides, that divide it, and of one slot."""
    new, lengths = {16: ((1, 1, 1), (700, 33, 1)), 32: ((12, 3, 17), (300, 64, 17)), 128: ((150, 40, 1), (700, 40, 90))}[rows]
    whole = d * (1 if states == INT8 else torch.finfo(TYPES[t]).bits // 8) % 16 == 0
    if states == SAME:
        kernel = ((32 if t == "f32" and rows < 128 else rows), 1 if rows < 128 else 4, WHOLE) if whole else (32, 1, LOOSE)
    elif rows == 128:
        kernel = (128, 4, CODES)
    else:
        kernel = (rows, 1, BYTES) if whole and t != "f32" else (32, 1, CODES)
    assert O.self_kernel(sum(new), 3, 4, 2, d, TYPES[t], states, whole) == kernel
    kept = ONCE[t] if kernel[1] == 4 else TWO[t]
    q = rows_of(d, sum(new), 4, d, t)
    for page in (16, 64, 24, 1):
        cache = Cache(d + page, new, lengths, 2, d, t, "same" if states == SAME else "i8", page)
        for window in (0, 5, 70):
            check_cache(cache, q, attend(context, cache, q, window), kept, window)


@pytest.mark.parametrize("heads, d", [(8, 64), (40, 64), (8, 40)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_weights_over_int8_values_are_the_sum_of_their_numbers(context, heads, d, t):
    """Few states a row and many rows: tens of thousands of weights times scales, some of them next to the border of two
    numbers, where the first number and what it leaves have to be of the same product."""
    n = 500
    cache = Cache(d, (1,) * n, (8,) * n, 2, d, t, "i8", 8)
    q = rows_of(1, n, heads, d, t)
    out = attend(context, cache, q)
    k, v, sv = (torch.stack([f(cache.at(i, 0, 8)) for i in range(n)]) for f in
                (lambda at: cache.values(0, at), lambda at: cache.values(1, at), lambda at: cache.scales[1][at].double()))
    # (A sequence's rows see all of its states: heads as rows of one product.)
    qs = q.double().view(n, 2, heads // 2, d)
    kk, vv = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    s = torch.matmul(qs, kk) * d ** -0.5
    pr = torch.softmax(s, -1)
    want = torch.matmul(pr, vv)
    a = torch.matmul(qs.abs(), kk.abs()).amax(-1, keepdim=True) * d ** -0.5
    off = 2 * ((d + 6) * 2.0 ** -24 * a + 2.0 ** -22 * s.abs().amax(-1, keepdim=True)) + 2.0 ** -21 + 8 * 2.0 ** -23 + TWO[t]
    half, tiny = torch.finfo(q.dtype).eps / 2, torch.finfo(q.dtype).tiny
    tol = torch.matmul(pr * off, vv.abs()) * 1.01 + want.abs().clamp_min(tiny) * half * 1.01
    if t == "f16":
        tol = tol + 1.01 * 2.0 ** -25 * pr.amax(-1, keepdim=True) * 127 * 8 * 4 * sv.amax(1)[:, :, None, None]
    worst = ((out.double().view_as(want) - want).abs() / tol).max().item()
    assert worst <= 1, worst
