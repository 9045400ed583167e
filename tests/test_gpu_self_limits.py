"""Attention of a call's own tokens and the rows of its cache at the ends of their ranges, on an MI355X: very long
sequences, very many key heads, strides at the border of 31 bits, lengths past everything, slots that come and go."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import turboembed_amd as T  # noqa: E402
from paged import TYPES, Cache, ints, starts_of, stream  # noqa: E402
from test_gpu_self_kernels import ONCE, TWO, attend, check, check_cache, check_prompt, prompt, rows_of  # noqa: E402
from test_self_kernels import CHUNKS, LOOSE  # noqa: E402
from turboembed_amd import operators as O  # noqa: E402


@pytest.mark.parametrize("t, n, d", [("bf16", 70001, 64), ("f16", 65000, 64), ("f32", 33000, 40), ("f32", 66001, 32)])
def test_a_prompt_of_very_many_tokens(context, t, n, d):
    """One sequence: its first rows, its last ones, and some between."""
    q, k, v = rows_of(1, n, 1, d, t), rows_of(2, n, 1, d, t), rows_of(3, n, 1, d, t)
    kept = ONCE[t] if O.self_kernel(n, 1, 1, 1, d, TYPES[t])[0] == 128 else TWO[t]
    for window in (0, 1000):
        out = torch.full_like(q, 3.0)
        context.prompt_attention(q, k, v, starts_of([n]), out, window=window, stream=stream())
        for a in (0, 4000, n // 2, n - 70):
            check(out[a:a + 70], q[a:a + 70], a, k[:a + 70].double(), v[:a + 70].double(), kept, window)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("t, held", [("bf16", "same"), ("f16", "i8"), ("f32", "same")])
def test_a_token_over_very_many_states(context, t, held):
    n = (1 << 20) + 37
    cache = Cache(1, (2,), (n,), 1, 64, t, held, 64)
    q = rows_of(2, 2, 8, 64, t)
    for window in (0, 70000):
        check_cache(cache, q, attend(context, cache, q, window), TWO[t], window)


@pytest.mark.parametrize("kv", [300, 1000, 4000])
@pytest.mark.parametrize("t, held", [("bf16", "same"), ("f16", "i8"), ("f32", "same")])
def test_very_many_key_heads(context, kv, t, held):
    cache = Cache(1, (1, 2, 9), (90, 2, 40), kv, 16, t, held, 16)
    q = rows_of(2, 12, 2 * kv, 16, t)
    check_cache(cache, q, attend(context, cache, q), TWO[t])
    n = 90
    q, k, v = rows_of(n, n, 2 * kv, 16, t), rows_of(n + 1, n, kv, 16, t), rows_of(n + 2, n, kv, 16, t)
    prompt(context, q, k, v, (60, 30), ONCE[t])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_blocks_within_a_token_s_heads(context, t):
    """200 heads to a key head, in the kernels of long prompts."""
    q, k, v = rows_of(1, 71, 1600, 32, t), rows_of(2, 71, 8, 32, t), rows_of(3, 71, 8, 32, t)
    assert O.self_kernel(71, 2, 1600, 8, 32, TYPES[t]) == ((32, 1, CHUNKS) if t == "f32" else (128, 4, CHUNKS))
    for window in (0, 9):
        prompt(context, q, k, v, (41, 30), ONCE[t], window)


@pytest.mark.parametrize("step, held", [((1 << 23) - 64, CHUNKS), (1 << 23, LOOSE)])
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_prompts_of_strides_around_31_bits(context, step, held, t):
    """Tiles whose bytes 31 bits hold go as whole chunks, others through registers."""
    n, d = 200, 64
    pool = torch.zeros(n * step + 1024, dtype=TYPES[t], device="cuda")
    q, k, v, out = (pool.as_strided((n, 1, d), (step, d, 1), at) for at in (0, 128, 256, 384))
    for i, x in enumerate((q, k, v)):
        x.copy_(rows_of(i, n, 1, d, t))
    context.prompt_attention(q, k, v, starts_of([150, 50]), out, stream=stream())
    check_prompt(out, q, k, v, (150, 50), TWO[t])


def test_cache_rows_of_more_than_a_launch(context):
    """More rows than 2^20 workgroups of 64 take at once."""
    n, page = (1 << 26) + 1000, 1 << 16
    columns = (n + page - 1) // page
    pages = torch.randperm(columns, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()[None]
    k = torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 1, 2).to(torch.int16).view(torch.float16)
    v = (7 * torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 1, 2)).to(torch.int16).view(torch.float16)
    ck, cv = (torch.zeros(columns * page, 1, 2, dtype=torch.float16, device="cuda") for _ in "kv")
    cache, arrays = T.StateCache(ck, cv, page), (starts_of([n]), ints([n]), pages)
    context.cache_write(k, v, cache, *arrays, stream=stream())
    for x, c in ((k, ck), (v, cv)):
        got = c.view(columns, page, 2)[pages[0].long()].view(-1, 2)[:n]
        same = torch.equal(got.view(torch.int16), x.view(n, 2).view(torch.int16))
        assert same
    gk, gv = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    context.cache_read(cache, *arrays, gk, gv, stream=stream())
    for x, y in ((k, gk), (v, gv)):
        same = torch.equal(x.view(torch.int16), y.view(torch.int16))
        assert same


@pytest.mark.parametrize("t, held", [("bf16", "same"), ("f16", "i8"), ("f32", "i8")])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_lengths_past_everything(context, t, held, m):
    """A length of 2^31 - 1: every state that the pages hold is seen, or, with a window, none."""
    n = 240
    cache = Cache(1, (m, 1), (n, 9), 2, 64, t, held, 16)
    cache.lengths.copy_(ints([2147483647, 9]))
    q = rows_of(2, m + 1, 4, 64, t)
    kept = ONCE[t] if 2 * (m + 1) > 64 else TWO[t]
    for window in (0, 2147483647, 1 << 30, 70):
        out = attend(context, cache, q, window)
        where = cache.at(0, 0, n)
        unit = 4 * cache.scales[1][where].amax().double() * torch.ones(m, 1, device="cuda") if held == "i8" else None
        if window in (70, 1 << 30):
            assert (out[:m] == 0).all()
        else:
            check(out[:m], q[:m], n, cache.values(0, where), cache.values(1, where), kept, unit=unit)
        where = cache.at(1, 0, 9)
        unit = 4 * cache.scales[1][where].amax().double() * torch.ones(1, 1, device="cuda") if held == "i8" else None
        check(out[m:], q[m:], 8, cache.values(0, where), cache.values(1, where), kept, window, unit=unit)


@pytest.mark.parametrize("held", ["same", "i8"])
def test_a_captured_step_whose_sequences_come_and_go(context, held):
    """One graph of write, attention and read: each replay has other sequences with a token, a chunk, or none, as `starts`
    says; rows that are nobody's are left."""
    t, kv, d, page, tokens = "bf16", 2, 64, 16, 64
    lens = [300, 90, 40, 700, 16, 33, 128, 64]
    cache = Cache(3, (0,) * 8, lens, kv, d, t, held, page)
    q, k, v = rows_of(1, tokens, 4, d, t), rows_of(2, tokens, kv, d, t), rows_of(3, tokens, kv, d, t)
    out, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = torch.empty(context.cache_workspace(tokens, 8, 4, kv, d, TYPES[t]), dtype=torch.uint8, device="cuda")
    operand, arrays = cache.operand(T), cache.arrays()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        context.cache_write(k, v, operand, *arrays, stream=stream())
        context.cache_attention(q, operand, *arrays, out, workspace=ws, stream=stream())
        context.cache_read(operand, *arrays, gk, gv, stream=stream())
    for step, rows in enumerate(((1,) * 8, (0, 0, 1, 0, 0, 0, 0, 1), (0,) * 8, (1, 0, 40, 1, 0, 16, 1, 1), (0, 0, 0, 64, 0, 0, 0, 0),
                                 (1,) * 8)):
        for x, seed in ((q, 10), (k, 20), (v, 30)):
            x.copy_(rows_of(seed + step, tokens, x.shape[1], d, t))
        cache.rows = rows
        cache.starts.copy_(starts_of(rows))
        n = sum(rows)
        for x in (out, gk, gv):
            x.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = TWO[t]       # (128 rows of 8 sequences: blocks of 16)
        check_cache(cache, q, out, kept)
        if n:
            slots = cache.new_slots()
            for i, (x, got) in enumerate(((k, gk), (v, gv))):
                held_now = cache.values(i, slots)
                same = torch.equal(got[:n].double(), held_now.to(torch.bfloat16).double())
                assert same
                if held == "same":
                    same = torch.equal(got[:n], x[:n])
                    assert same
                else:
                    top = x[:n].double().abs().amax(-1, keepdim=True)
                    assert ((held_now - x[:n].double()).abs() <= top / 253).all()
        for x in (out, gk, gv):
            assert (x[n:] == 3).all()
