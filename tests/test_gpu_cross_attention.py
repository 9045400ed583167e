"""Attention of queries to an encoder's states of another length, on an MI355X against 64-bit arithmetic on the same
inputs.

Tolerance, from the roundings that the operator states. A score is a sum of `width` F32 products in some order, times a
factor and less a maximum: off by at most e = (width + 4) 2^-24 A + 2^-22 S, A the largest sum of |q_c k_c| scale and S
the largest |score| of the row. A probability is then off by a factor of 1 +- (2 e + 2^-21) against its row's sum, by
half a step of the type where it is rounded to it (16-bit operands), and, in F16, by half a step of the smallest number,
2^-25 of the row's largest. The products with V are summed in F32 in some order, n 2^-24 each, and the output is rounded
once."""
import math

import pytest

import turboembed_amd as T
from turboembed_amd import seam as S

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _workspace(plan):
    # (Whatever it holds: nothing is kept in it between calls.)
    return torch.full((plan.workspace_bytes,), 0xff, dtype=torch.uint8, device="cuda")


def _operands(seed, nq, nk, heads, kv, d, t, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: (torch.randn(*s, generator=g) * spread).to(TYPES[t]).cuda()  # noqa: E731
    return f(nq, heads, d), f(nk, kv, d), f(nk, kv, d)


def _check(out, q, k, v, q_lens, k_lens, mask=None, scale=None):
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    half = torch.finfo(out.dtype).eps / 2
    tiny = torch.finfo(out.dtype).tiny
    f32 = out.dtype == torch.float32
    qat = kat = 0
    for nq, nk in zip(q_lens, k_lens):
        keep = torch.arange(kat, kat + nk, device="cuda")
        if mask is not None:
            keep = keep[mask[kat:kat + nk] != 0]
        qs, o = q[qat:qat + nq].double(), out[qat:qat + nq].double()
        ks, vs = (x[keep].double().repeat_interleave(heads // kv, 1) for x in (k, v))
        qat, kat = qat + nq, kat + nk
        if nq == 0:
            continue
        if len(keep) == 0:
            assert (o == 0).all()
            continue
        s = torch.matmul(qs.transpose(0, 1), ks.permute(1, 2, 0)) * scale
        p = torch.softmax(s, -1)
        want = torch.matmul(p, vs.transpose(0, 1)).transpose(0, 1)
        a = torch.matmul(qs.abs().transpose(0, 1), ks.abs().permute(1, 2, 0)).amax(-1, keepdim=True) * abs(scale)
        e = (d + 4) * 2.0 ** -24 * a + 2.0 ** -22 * s.abs().amax(-1, keepdim=True)
        off = 2 * e + 2.0 ** -21 + len(keep) * 2.0 ** -23 + (0 if f32 else half)
        weight = torch.matmul(p * off, vs.abs().transpose(0, 1)).transpose(0, 1)
        if out.dtype == torch.float16:
            weight = weight + 2.0 ** -25 * (p.amax(-1) .transpose(0, 1)[..., None] * vs.abs().sum(0)[None])
        tol = weight * 1.01 + want.abs().clamp_min(tiny) * half * 1.01
        assert torch.isfinite(o).all()
        worst = ((o - want).abs() / tol).max().item()
        assert worst <= 1, (nq, nk, worst)


def _run(context, q_lens, k_lens, heads, kv, d, t, seed=0, mask=None, scale=None, spread=1.0):
    q, k, v = _operands(seed, sum(q_lens), sum(k_lens), heads, kv, d, t, spread)
    out = torch.full_like(q, 3.0)
    plan = context.cross_plan(q_lens, k_lens, heads, kv, d, TYPES[t])
    plan.run(q, k, v, out, mask=mask, scale=scale, workspace=_workspace(plan), stream=_stream())
    _check(out, q, k, v, q_lens, k_lens, mask, scale)
    plan.close()


LENGTHS = [
    ((1,), (1,)), ((1,), (31,)), ((1,), (33,)), ((1, 1, 1), (64, 1, 200)), ((2,), (65,)), ((1,) * 9, (7,) * 9),
    ((1,), (3000,)), ((5,), (1025,)), ((16, 3), (300, 17)), ((32,), (32,)), ((33, 1, 70), (63, 129, 64)),
    ((128,), (128,)), ((129, 0, 4), (257, 5, 0)), ((200, 7), (1, 511)), ((300,), (700,))]


@pytest.mark.parametrize("q_lens, k_lens", LENGTHS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads, kv, d", [(1, 1, 64), (6, 2, 64), (4, 4, 32), (8, 1, 128), (3, 3, 80)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_cross_attention_is_the_formula_s(context, q_lens, k_lens, heads, kv, d, t):
    _run(context, q_lens, k_lens, heads, kv, d, t, seed=sum(q_lens) + sum(k_lens))


@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 9, 16, 24, 31, 33, 40, 48, 63, 65, 72, 96, 100, 112, 127])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_every_kind_of_head_width(context, d, t):
    _run(context, (1, 1), (40, 90), 2, 1, d, t, seed=d)
    _run(context, (50, 9), (40, 90), 2, 2, d, t, seed=d)


@pytest.mark.parametrize("q_lens", [(1, 1, 1, 1, 1), (3, 1, 40, 5, 9), (130, 20, 1, 64, 300)])
@pytest.mark.parametrize("d", [32, 64, 72])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_masked_states_and_sequences_with_none(context, q_lens, d, t):
    k_lens = (70, 300, 33, 1, 513)
    q, k, v = _operands(d, sum(q_lens), sum(k_lens), 4, 2, d, t)
    g = torch.Generator().manual_seed(d)
    mask = (torch.rand(sum(k_lens), generator=g) < 0.6).to(torch.int32).cuda()
    mask[70:370] = 0                    # the second sequence has nothing live
    mask[370 + 1:370 + 33] = 0          # the third one state, its first
    mask[370] = -5                      # (any entry but 0)
    mask[404 + 128:404 + 448] = 0       # a stretch of whole tiles
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(TYPES[t]).min):
        kk, vv = k.clone(), v.clone()
        kk[mask == 0] = junk
        vv[mask == 0] = junk
        out = torch.full_like(q, 3.0)
        plan = context.cross_plan(q_lens, k_lens, 4, 2, d, TYPES[t])
        plan.run(q, kk, vv, out, mask=mask, workspace=_workspace(plan), stream=_stream())
        _check(out, q, kk, vv, q_lens, k_lens, mask)
        plan.close()


@pytest.mark.parametrize("nq", [1, 6, 150])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_the_states_of_a_neighbour_are_not_seen(context, nq, t):
    # The sequences before and after, and what lies behind the last, hold no numbers.
    q, k, v = _operands(1, 3 * nq, 300, 2, 2, 64, t)
    k[:37] = v[:37] = float("nan")
    k[137:] = v[137:] = float("inf")
    q_lens, k_lens = (nq, nq, nq), (37, 100, 63)
    out = torch.full((3 * nq + 2, 2, 64), 3.0, dtype=TYPES[t], device="cuda")
    plan = context.cross_plan(q_lens, k_lens, 2, 2, 64, TYPES[t])
    plan.run(torch.cat([q, q[:2]]), k, v, out, workspace=_workspace(plan), stream=_stream())
    _check(out[nq:2 * nq], q[nq:2 * nq], k[37:137], v[37:137], (nq,), (100,))
    assert (out[3 * nq:] == 3).all()     # rows behind the last sequence


@pytest.mark.parametrize("nq", [1, 3, 90])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_layouts(context, nq, t):
    heads, kv, d, nk = 4, 2, 64, 333
    q, k, v = _operands(2, nq, nk, heads, kv, d, t)
    plan = context.cross_plan((nq,), (nk,), heads, kv, d, TYPES[t])
    ws = _workspace(plan)

    def run(q, k, v, out):
        plan.run(q, k, v, out, workspace=ws, stream=_stream())
        _check(out, q, k, v, (nq,), (nk,))
        return out
    plain = run(q, k, v, torch.empty_like(q))
    # Head by head; keys and values side by side; columns of wider rows that start at any element.
    hm = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    assert torch.equal(plain, run(hm(q), hm(k), hm(v), hm(torch.empty_like(q))))
    both = torch.stack([k, v], 1)
    assert torch.equal(plain, run(q, both[:, 0], both[:, 1], torch.empty_like(q)))

    def loose(x, off):
        wide = torch.full((x.shape[0], x.shape[1] * d + 13), 2.0, dtype=x.dtype, device="cuda")
        y = wide[:, off:off + x.shape[1] * d].unflatten(1, (x.shape[1], d))
        y.copy_(x)
        return wide, y
    wide, out = loose(torch.empty_like(q), 5)
    assert torch.equal(plain, run(loose(q, 1)[1], loose(k, 3)[1], loose(v, 7)[1], out))
    assert (wide[:, :5] == 2).all() and (wide[:, 5 + heads * d:] == 2).all()
    # One state for all, and one query.
    run(q[:1].expand(nq, heads, d), k, v, torch.empty_like(q))
    run(q, k[:1].expand(nk, kv, d), v[:1].expand(nk, kv, d), torch.empty_like(q))
    # One key head for all heads (stride 0).
    run(q, k[:, :1].expand(nk, kv, d), v[:, :1].expand(nk, kv, d), torch.empty_like(q))
    plan.close()


@pytest.mark.parametrize("nq", [1, 5, 100])
@pytest.mark.parametrize("scale", [0.0, -0.5, 1.0, 1e-30])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scales(context, nq, scale, t):
    _run(context, (nq,), (257,), 2, 2, 64, t, scale=scale)


@pytest.mark.parametrize("nq", [1, 5, 100])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_scores_far_apart_and_far_from_zero(context, nq, t):
    # Scores of some 1e12: one state takes all, exactly.
    q, k, v = _operands(4, nq, 200, 2, 2, 64, t)
    q, k = q.abs() * 1e6, k * 1e5
    out = torch.empty_like(q)
    plan = context.cross_plan((nq,), (200,), 2, 2, 64, TYPES[t])
    plan.run(q, k, v, out, workspace=_workspace(plan), stream=_stream())
    s = torch.matmul(q.double().transpose(0, 1), k.double().permute(1, 2, 0))
    two = s.topk(2, -1)
    gap = two.values[..., 0] - two.values[..., 1]
    sure = gap > 1e-5 * two.values.abs().amax(-1) + 1e3           # [heads, nq]
    assert sure.float().mean() > 0.8
    best = torch.gather(v.transpose(0, 1), 1, two.indices[..., :1].expand(-1, -1, 64))
    assert torch.equal(out.transpose(0, 1)[sure], best[sure])
    plan.close()


@pytest.mark.parametrize("nq", [1, 5, 100])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scores_that_are_infinite_or_not_numbers(context, nq, t):
    q, k, v = _operands(5, nq, 150, 1, 1, 64, t)
    q[:, :, 0] = 1.0
    plan = context.cross_plan((nq,), (150,), 1, 1, 64, TYPES[t])
    mask = torch.ones(150, dtype=torch.int32, device="cuda")
    mask[70:] = 0

    def run(k, mask=None):
        out = torch.empty_like(q)
        plan.run(q, k, v, out, mask=mask, workspace=_workspace(plan), stream=_stream())
        return out
    for at in (3, 149):
        for bad in (float("nan"), float("inf")):
            kk = k.clone()
            kk[at, 0, 0] = bad
            assert torch.isnan(run(kk)).all()
        # A state whose score is minus infinity weighs nothing.
        kk = k.clone()
        kk[at, 0, 0] = -float("inf")
        keep = torch.arange(150, device="cuda") != at
        _check(run(kk), q, torch.where(keep[:, None, None], kk, 0), v, (nq,), (150,), keep.to(torch.int32))
    # All of them: what the softmax of minus infinities is.
    kk = k.clone()
    kk[:, 0, 0] = -float("inf")
    assert torch.isnan(run(kk)).all() and torch.isnan(run(kk, mask)).all()
    # A live value that is infinite is what its product gives.
    vv = v.clone()
    v = vv
    v[7, 0, 5] = float("inf")
    o = run(k)
    assert (o[:, 0, 5] == float("inf")).all() and torch.isfinite(o[:, 0, :5]).all()
    plan.close()


def test_nothing_to_do(context):
    for q_lens, k_lens in (((), ()), ((0, 0), (5, 0)), ((0,), (0,))):
        q, k, v = _operands(0, 0, sum(k_lens), 2, 2, 32, "f16")
        plan = context.cross_plan(q_lens, k_lens, 2, 2, 32, torch.float16)
        plan.run(q, k, v, torch.empty_like(q), workspace=_workspace(plan), stream=_stream())
        plan.close()
    # No states at all: zeros.
    q, k, v = _operands(0, 7, 0, 2, 2, 32, "bf16")
    out = torch.full_like(q, 4.0)
    plan = context.cross_plan((3, 4), (0, 0), 2, 2, 32, torch.bfloat16)
    plan.run(q, k, v, out, workspace=_workspace(plan), stream=_stream())
    assert (out == 0).all()
    plan.close()


def test_a_workspace_too_small_is_refused(context):
    plan = context.cross_plan((1,), (20000,), 2, 2, 64, torch.float16)
    assert plan.workspace_bytes > 0     # one token against many states: its keys are cut
    q, k, v = _operands(0, 1, 20000, 2, 2, 64, "f16")
    out = torch.empty_like(q)
    ws = torch.empty(plan.workspace_bytes + 16, dtype=torch.uint8, device="cuda")
    for bad in (None, ws[:plan.workspace_bytes - 1]):
        with pytest.raises(T.TurboError) as e:
            plan.run(q, k, v, out, workspace=bad, stream=_stream())
        assert e.value.code == S.TURBO_E_CAPACITY
    for bad in (ws[1:], k.view(torch.uint8).flatten()[:plan.workspace_bytes + 16]):
        with pytest.raises(T.TurboError) as e:
            plan.run(q, k, v, out, workspace=bad, stream=_stream())
        assert e.value.code == S.TURBO_E_INVALID_ARGUMENT
    plan.run(q, k, v, out, workspace=ws)          # the context's own stream, waited for
    _check(out, q, k, v, (1,), (20000,))
    plan.close()


@pytest.mark.parametrize("q_lens, k_lens", [((1, 1), (900, 20000)), ((40, 9), (300, 5000)), ((300,), (1000,))])
def test_captured_and_replayed_beside_another(context, q_lens, k_lens):
    t, heads, kv, d = "bf16", 4, 2, 64
    plan = context.cross_plan(q_lens, k_lens, heads, kv, d, TYPES[t])
    calls = []
    for seed in range(2):
        q, k, v = _operands(seed, sum(q_lens), sum(k_lens), heads, kv, d, t)
        out, ws = torch.empty_like(q), _workspace(plan)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan.run(q, k, v, out, workspace=ws, stream=_stream())
        calls.append((q, k, v, out, g, torch.cuda.Stream()))
    for again in range(4):
        for q, k, v, out, g, s in calls:
            q.copy_(_operands(10 + again, sum(q_lens), sum(k_lens), heads, kv, d, t)[0])
            out.zero_()
        torch.cuda.synchronize()
        # One plan, two graphs, two streams.
        for *_, g, s in calls:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for q, k, v, out, _, _ in calls:
            _check(out, q, k, v, q_lens, k_lens)
    plan.close()


@pytest.mark.parametrize("q_lens, k_lens", [((1,), (5000,)), ((30,), (3000,)), ((500,), (400,))])
def test_the_same_call_gives_the_same_bits(context, q_lens, k_lens):
    q, k, v = _operands(8, sum(q_lens), sum(k_lens), 2, 2, 64, "f16")
    plan = context.cross_plan(q_lens, k_lens, 2, 2, 64, torch.float16)
    outs = []
    for _ in range(5):
        out = torch.empty_like(q)
        plan.run(q, k, v, out, workspace=_workspace(plan), stream=_stream())
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs)
    plan.close()


def test_offsets_past_32_bits(context):
    # States further apart than 2^32 bytes reach: one head's columns of wide rows.
    heads, d, nk = 1, 64, 600
    step = 4 * 1024 * 1024       # elements; 600 rows of them are 4.7 GiB of 16-bit values
    wide = torch.empty(nk * step, dtype=torch.float16, device="cuda")
    k = wide.as_strided((nk, heads, d), (step, d, 1))
    v = wide.as_strided((nk, heads, d), (step, d, 1), 128)
    kk, vv = _operands(6, 1, nk, heads, heads, d, "f16")[1:]
    k.copy_(kk)
    v.copy_(vv)
    for nq in (1, 64):
        q = _operands(7, nq, 1, heads, heads, d, "f16")[0]
        out = torch.empty_like(q)
        plan = context.cross_plan((nq,), (nk,), heads, heads, d, torch.float16)
        plan.run(q, k, v, out, workspace=_workspace(plan), stream=_stream())
        _check(out, q, kk, vv, (nq,), (nk,))
        plan.close()


def _codes(context, x):
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    k = torch.empty(x.shape[0], device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    return q, k


def test_a_sublayer_over_a_session_s_states(context):
    """Norm, int8 products, attention to an encoder's states, its rows' codes, the output product, the next norm: as a
    reader of a session's hidden states runs them, once eagerly and from a graph, against the same steps in 64 bits on
    the codes that were made."""
    import small
    from test_gpu_row_codes import _close
    desc = small.bert(seed=5, hidden=96, heads=3, inter=64)
    model = context.load(desc)
    s = model.session(4, 24, S.TURBO_PRECISION_EXACT)
    import numpy as np
    g = np.random.Generator(np.random.PCG64(1))
    ids = g.integers(3, desc.vocab_size - 1, size=(4, 24)).astype(np.int32)
    lens = [24, 7, 1, 15]
    mask = (np.arange(24)[None] < np.array(lens)[:, None]).astype(np.int32)
    s.embed(ids, mask)
    states = torch.from_numpy(s.hidden()).cuda()
    s.close()
    model.close()
    hidden, heads, d, q_lens = 96, 3, 32, [5, 1, 3, 2]
    n = sum(q_lens)
    g = torch.Generator().manual_seed(2)
    f = lambda *z: torch.randn(*z, generator=g).cuda()  # noqa: E731
    stream, update = f(n, hidden), f(n, hidden).half()
    w1, w2 = 1 + 0.1 * f(hidden), 1 + 0.1 * f(hidden)
    wq, wkv, wo = (_codes(context, f(r, hidden) / hidden ** 0.5) for r in (hidden, 2 * hidden, hidden))
    bo = f(hidden)
    new = lambda *z, t=torch.float16: torch.empty(*z, dtype=t, device="cuda")  # noqa: E731
    total, c1, s1 = new(n, hidden, t=torch.float32), new(n, hidden, t=torch.int8), new(n, t=torch.float32)
    q, cs, ss = new(n, hidden), new(sum(lens), hidden, t=torch.int8), new(sum(lens), t=torch.float32)
    kv, ctx = new(sum(lens), 2 * hidden), new(n, heads, d)
    c2, s2, o = new(n, hidden, t=torch.int8), new(n, t=torch.float32), new(n, hidden)
    total2, y = new(n, hidden, t=torch.float32), new(n, hidden)
    plan = context.cross_plan(q_lens, lens, heads, heads, d, torch.float16)
    ws = _workspace(plan)

    def layer():
        at = _stream()
        context.rms_norm(update, w1, 1e-6, residual=stream, sum=total, codes=c1, scales=s1, stream=at)
        context.linear_i8(c1, s1, *wq, q, stream=at)
        context.quantize_tokens(states, cs, ss, stream=at)
        context.linear_i8(cs, ss, *wkv, kv, stream=at)
        k3, v3 = kv.view(-1, 2, heads, d)[:, 0], kv.view(-1, 2, heads, d)[:, 1]
        plan.run(q.view(n, heads, d), k3, v3, ctx, workspace=ws, stream=at)
        context.quantize_tokens(ctx.view(n, hidden), c2, s2, stream=at)
        context.linear_i8(c2, s2, *wo, o, bias=bo, stream=at)
        context.rms_norm(o, w2, 1e-6, residual=total, sum=total2, out=y, stream=at)
    layer()
    torch.cuda.synchronize()
    first = [t.clone() for t in (total, c1, q, kv, ctx, c2, o, total2, y)]

    def product(c, cs, w, b=0.0):
        return (c.double() @ w[0].double().T) * cs.double()[:, None] * w[1].double() + b
    # Each step on what the step before wrote: the output's rounding and a few F32 ones.
    def near(got, want, t):
        tol = want.abs().clamp_min(torch.finfo(t).tiny) * torch.finfo(t).eps / 2 + want.abs().amax() * 2.0 ** -20
        assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(total, update.float() + stream)
    near(q, product(c1, s1, wq), torch.float16)
    near(kv, product(cs, ss, wkv), torch.float16)
    _check(ctx, q.view(n, heads, d), kv.view(-1, 2, heads, d)[:, 0], kv.view(-1, 2, heads, d)[:, 1], q_lens, lens)
    near(o, product(c2, s2, wo, bo.double()), torch.float16)
    v = total2.double()
    assert torch.equal(total2, o.float() + total)
    _close(y, (v * w2.double() / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)).cpu().numpy(), "f16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for _ in range(3):
        for t in (total, c1, q, kv, ctx, c2, o, total2, y):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (total, c1, q, kv, ctx, c2, o, total2, y)))
    plan.close()


@pytest.mark.parametrize("step", [(1 << 23) - 8, 1 << 23])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_states_far_apart(context, step, t):
    """The longest strides that a tile's 32-bit offsets take, and the first that go another way."""
    heads, d, nk = 1, 64, 70
    wide = torch.empty(nk * step, dtype=TYPES[t], device="cuda")
    k = wide.as_strided((nk, heads, d), (step, d, 1))
    v = wide.as_strided((nk, heads, d), (step, d, 1), 128)
    kk, vv = _operands(8, 1, nk, heads, heads, d, t)[1:]
    k.copy_(kk)
    v.copy_(vv)
    for nq in (1, 64):
        q = _operands(9, nq, 1, heads, heads, d, t)[0]
        out = torch.empty_like(q)
        plan = context.cross_plan((nq,), (nk,), heads, heads, d, TYPES[t])
        plan.run(q, k, v, out, workspace=_workspace(plan), stream=_stream())
        _check(out, q, kk, vv, (nq,), (nk,))
        plan.close()
