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
