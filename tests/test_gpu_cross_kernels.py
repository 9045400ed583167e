"""Cross attention's kernels, each of them, on an MI355X against 64-bit arithmetic on the same inputs.

Tolerance: as for the operator (scores off by at most e = (width + 4) 2^-24 A + 2^-22 S, A the largest sum of
|q_c k_c| scale and S the largest |score| of the row; a probability by a factor of 1 +- (2 e + 2^-21) against its sum;
n 2^-24 and once more for the sums of n products; the output rounded once), but for the rounding of a 16-bit
probability p, which goes by the kernel. One number of the type: half a step, eps / 2. Two: the first is one to two
steps below p, the second what is left, at most 2 eps p, rounded: eps / 2 of that, so eps^2 p. In F16 besides half a
step of the smallest number, 2^-25 of the row's largest probability."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _operands(seed, nq, nk, heads, kv, d, t, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: (torch.randn(*s, generator=g) * spread).to(TYPES[t]).cuda()  # noqa: E731
    return f(nq, heads, d), f(nk, kv, d), f(nk, kv, d)


def _check(out, q, k, v, q_lens, k_lens, rounding, mask=None):
    """`rounding`: of a probability, relative to it."""
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    info = torch.finfo(out.dtype)
    qat = kat = 0
    for nq, nk in zip(q_lens, k_lens):
        keep = torch.arange(kat, kat + nk, device="cuda")
        if mask is not None:
            keep = keep[mask[kat:kat + nk] != 0]
        qs, o = q[qat:qat + nq].double(), out[qat:qat + nq].double()
        ks, vs = (x[keep].double().repeat_interleave(heads // kv, 1) for x in (k, v))
        qat, kat = qat + nq, kat + nk
        if nq == 0 or len(keep) == 0:
            assert (o == 0).all()
            continue
        s = torch.matmul(qs.transpose(0, 1), ks.permute(1, 2, 0)) * d ** -0.5
        p = torch.softmax(s, -1)
        want = torch.matmul(p, vs.transpose(0, 1)).transpose(0, 1)
        a = torch.matmul(qs.abs().transpose(0, 1), ks.abs().permute(1, 2, 0)).amax(-1, keepdim=True) * d ** -0.5
        e = (d + 4) * 2.0 ** -24 * a + 2.0 ** -22 * s.abs().amax(-1, keepdim=True)
        off = 2 * e + 2.0 ** -21 + len(keep) * 2.0 ** -23 + rounding
        weight = torch.matmul(p * off, vs.abs().transpose(0, 1)).transpose(0, 1)
        if out.dtype == torch.float16:
            weight = weight + 2.0 ** -25 * (p.amax(-1).transpose(0, 1)[..., None] * vs.abs().sum(0)[None])
        tol = weight * 1.01 + want.abs().clamp_min(info.tiny) * (info.eps / 2) * 1.01
        assert torch.isfinite(o).all()
        worst = ((o - want).abs() / tol).max().item()
        assert worst <= 1, (nq, nk, worst)


def _run(context, q_lens, k_lens, heads, kv, d, t, rounding, seed=0, spread=1.0):
    q, k, v = _operands(seed, sum(q_lens), sum(k_lens), heads, kv, d, t, spread)
    out = torch.full_like(q, 3.0)
    plan = context.cross_plan(q_lens, k_lens, heads, kv, d, TYPES[t])
    ws = torch.full((plan.workspace_bytes,), 0xff, dtype=torch.uint8, device="cuda")
    plan.run(q, k, v, out, workspace=ws, stream=_stream())
    _check(out, q, k, v, q_lens, k_lens, rounding)
    plan.close()


def lengths(n, most):
    """n lengths from `most` down to about half of it."""
    return [max(1, most - (i * 7) % max(1, most // 2)) for i in range(n)]


# Calls that reach every kernel: 16 bits or not, rows of a workgroup, whether its rows are one wave's or more, whether
# keys are cut and joined; then sequences, tokens of each, longest states, key heads, heads of each, width.
KERNELS = [
    (True, 32, True, False, 55, 1, 22, 16, 1, 32), (True, 32, True, False, 61, 1, 20, 12, 1, 64),
    (True, 32, True, True, 5, 1, 1266, 8, 1, 32), (True, 32, True, True, 2, 1, 2636, 8, 1, 64),
    (True, 32, True, True, 48, 1, 4096, 16, 1, 72), (True, 32, False, False, 52, 33, 330, 16, 1, 32),
    (True, 32, False, True, 10, 150, 723, 1, 1, 32), (True, 32, False, True, 2, 150, 1090, 2, 1, 64),
    (True, 32, False, True, 1, 150, 714, 4, 1, 96), (True, 32, False, True, 1, 33, 334, 8, 4, 128),
    (True, 128, False, False, 1, 33, 22, 1, 1, 32), (True, 128, False, False, 1, 33, 38, 1, 1, 64),
    (True, 128, False, False, 1, 40, 27, 1, 1, 96), (True, 128, False, False, 3, 40, 24, 2, 4, 128),
    (True, 128, False, True, 1, 33, 608, 1, 1, 32), (True, 128, False, True, 2, 70, 637, 1, 2, 64),
    (True, 128, False, True, 1, 33, 403, 1, 1, 96), (True, 128, False, True, 1, 33, 434, 1, 1, 128),
    (True, 128, True, False, 1, 1, 21, 1, 2, 32), (True, 128, True, False, 1, 1, 23, 1, 1, 64),
    (True, 128, True, False, 1, 1, 25, 1, 1, 96), (True, 128, True, False, 2, 3, 20, 2, 2, 128),
    (True, 128, True, True, 1, 1, 514, 1, 1, 32), (True, 128, True, True, 1, 1, 672, 1, 1, 64),
    (True, 128, True, True, 1, 1, 444, 1, 1, 96), (True, 128, True, True, 2, 4, 468, 1, 1, 128),
    (False, 32, True, False, 1, 1, 30, 1, 1, 32), (False, 32, True, False, 1, 1, 24, 1, 1, 64),
    (False, 32, True, False, 1, 1, 20, 1, 2, 96), (False, 32, True, False, 1, 1, 25, 1, 1, 128),
    (False, 32, True, True, 1, 1, 201, 1, 1, 32), (False, 32, True, True, 1, 1, 181, 1, 1, 64),
    (False, 32, True, True, 1, 1, 74, 1, 2, 96), (False, 32, True, True, 1, 1, 79, 1, 1, 128),
    (False, 32, False, False, 1, 33, 22, 1, 1, 32), (False, 32, False, True, 1, 33, 160, 1, 1, 64),
    (False, 128, False, False, 4, 33, 20, 16, 4, 32), (False, 128, False, False, 14, 33, 23, 16, 1, 64),
    (False, 128, False, False, 37, 33, 21, 8, 1, 96), (False, 128, False, False, 34, 33, 23, 8, 1, 128),
    (False, 128, False, True, 2, 33, 323, 12, 1, 32), (False, 128, False, True, 2, 33, 344, 12, 1, 64),
    (False, 128, False, True, 5, 33, 93, 16, 1, 96), (False, 128, False, True, 2, 33, 1282, 4, 1, 128),
    (False, 128, True, False, 24, 1, 22, 12, 1, 32), (False, 128, True, True, 8, 1, 161, 16, 1, 64)]
CALLS = [(t, c) for c in KERNELS for t in (("f16", "bf16") if c[0] else ("f32",))]


def _name(x):
    return x if isinstance(x, str) else "-".join(map(str, x[1:]))


def _rounding(t, rows, one_tile):
    """Of a probability by the kernel of these workgroups."""
    eps = torch.finfo(TYPES[t]).eps
    return 0.0 if t == "f32" else eps ** 2 if rows == 32 or one_tile else eps / 2


@pytest.mark.parametrize("t, call", CALLS, ids=_name)
def test_every_kernel(context, t, call):
    """Each with keys and values that are whole aligned chunks and with rows that start at any element, with a mask
    (nothing live in one sequence, no numbers in masked places) and without, and with an infinite live value."""
    _, rows, one_tile, _, n, nq, most, kv, share, d = call
    q_lens, k_lens, heads = [nq] * n, lengths(n, most), kv * share
    rounding = _rounding(t, rows, one_tile)
    q, k, v = _operands(most + d, sum(q_lens), sum(k_lens), heads, kv, d, t)
    g = torch.Generator().manual_seed(d)
    mask = (torch.rand(sum(k_lens), generator=g) < 0.7).to(torch.int32).cuda()
    mask[0] = 1
    if n > 1:
        mask[k_lens[0]:k_lens[0] + k_lens[1]] = 0
    plan = context.cross_plan(q_lens, k_lens, heads, kv, d, TYPES[t])

    def run(k, v, mask=None):
        out = torch.full_like(q, 3.0)
        ws = torch.full((plan.workspace_bytes,), 0xff, dtype=torch.uint8, device="cuda")
        plan.run(q, k, v, out, mask=mask, workspace=ws, stream=_stream())
        return out

    def loose(x):
        wide = torch.full((x.shape[0], kv * d + 1), float("nan"), dtype=x.dtype, device="cuda")
        y = wide[:, 1:].unflatten(1, (kv, d))
        y.copy_(x)
        return y
    plain = run(k, v)
    _check(plain, q, k, v, q_lens, k_lens, rounding)
    assert torch.equal(plain, run(loose(k), loose(v)))
    assert torch.equal(plain, run(k, v))
    dead = mask == 0
    kk, vv = k.clone(), v.clone()
    kk[dead] = float("nan")
    vv[dead] = float("nan")
    masked = run(kk, vv, mask)
    _check(masked, q, k, v, q_lens, k_lens, rounding, mask)
    assert torch.equal(masked, run(loose(kk), loose(vv), mask))
    vv[0, 0, d - 1] = float("inf")
    for o in (run(kk, vv, mask), run(loose(kk), loose(vv), mask)):
        assert (o[:nq, :share, d - 1] == float("inf")).all()
        o[:nq, :share, d - 1] = masked[:nq, :share, d - 1]
        assert torch.equal(o, masked)
    plan.close()


@pytest.mark.parametrize("t, call", [("bf16", KERNELS[4]), ("f16", KERNELS[2]), ("f16", KERNELS[0]), ("bf16", KERNELS[25]),
                                     ("f32", KERNELS[31]), ("f32", KERNELS[42])], ids=_name)
def test_captured_and_replayed(context, t, call):
    _, rows, one_tile, _, n, nq, most, kv, share, d = call
    q_lens, k_lens, heads = [nq] * n, lengths(n, most), kv * share
    q, k, v = _operands(0, sum(q_lens), sum(k_lens), heads, kv, d, t)
    plan = context.cross_plan(q_lens, k_lens, heads, kv, d, TYPES[t])
    ws = torch.full((plan.workspace_bytes,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, k, v, out, workspace=ws, stream=_stream())
    for seed in range(3):
        for x, y in zip((q, k, v), _operands(seed + 1, sum(q_lens), sum(k_lens), heads, kv, d, t)):
            x.copy_(y)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, q_lens, k_lens, _rounding(t, rows, one_tile))
    plan.close()


@pytest.mark.parametrize("spread", [1.0, 2.0])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_one_token_s_probabilities_are_two_numbers(context, t, d, spread):
    """A token each of many sequences: nothing but the output's rounding shows."""
    n = 48
    k_lens = [200 + 83 * i for i in range(n)]
    _run(context, [1] * n, k_lens, 16, 16, d, t, torch.finfo(TYPES[t]).eps ** 2, seed=d, spread=spread)


@pytest.mark.parametrize("q_lens, k_lens", [((1,), (300,)), ((3, 40), (300, 250)), ((1,) * 40, (300,) * 40),
                                            ((200,), (300,)), ((1,), (3000,))])
@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("low", ["first", "every other 32"])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_values_as_large_as_their_sums_allow(context, t, low, direct, q_lens, k_lens):
    """Some states' scores are 0, those of others after them just under 8 in base 2, so that weights reach 2^8 where the
    maximum is that of the first; times the number of states the largest value is just what F32 holds.

    All values are positive: a relative error. Scores are exact; weights are off by 2^-21, sums of n by n 2^-23, a
    16-bit weight and the output by half a step each."""
    d, heads, most = 64, 2, max(k_lens)
    top = min(3.3e38 / most, 65000.0 if t == "f16" else 3e38)
    g = torch.Generator().manual_seed(most)
    step = d if direct else d + 1     # (rows that start at any element go another way)
    wide = torch.zeros(2, sum(k_lens), heads * step, dtype=TYPES[t])
    k, v = (wide[i].unflatten(1, (heads, step))[..., :d] for i in range(2))
    at = 0
    for n in k_lens:
        j = torch.arange(n)
        k[at:at + n, :, 0] = torch.where(j >= 70 if low == "first" else j % 64 >= 32, 7.875, 0.0)[:, None].to(k.dtype)
        at += n
    v.copy_(top * (0.25 + 0.75 * torch.rand(sum(k_lens), heads, d, generator=g).double()))
    wide = wide.cuda()
    k, v = (wide[i].unflatten(1, (heads, step))[..., :d] for i in range(2))
    q = torch.zeros(sum(q_lens), heads, d, dtype=TYPES[t], device="cuda")
    q[..., 0] = 1
    out = torch.empty_like(q)
    plan = context.cross_plan(q_lens, k_lens, heads, heads, d, TYPES[t])
    ws = torch.full((plan.workspace_bytes,), 0xff, dtype=torch.uint8, device="cuda")
    plan.run(q, k, v, out, scale=0.6931471805599453, workspace=ws, stream=_stream())
    plan.close()
    half = torch.finfo(TYPES[t]).eps / 2
    qat = kat = 0
    for nq, nk in zip(q_lens, k_lens):
        p = torch.softmax(k[kat:kat + nk, :, 0].double() * 0.6931471805599453, 0)
        want = (p[..., None] * v[kat:kat + nk].double()).sum(0)
        o = out[qat:qat + nq].double()
        qat, kat = qat + nq, kat + nk
        tol = want * (2.0 ** -20 + nk * 2.0 ** -23 + half + (0 if t == "f32" else half)) * 1.01
        assert ((o - want).abs() <= tol).all()
