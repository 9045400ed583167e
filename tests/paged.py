"""Caches of states in pages, and attention over them in 64 bits, for the tests of the operators that use them."""
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(rows):
    s = [0]
    for m in rows:
        s.append(s[-1] + m)
    return ints(s)


class Cache:
    """Sequences of `lengths` states, of which the last `rows` are a call's, in pages in no order; held: "same" or "i8".

    Slots that hold no state are full of NaN (of I8 states: their scales)."""

    def __init__(self, seed, rows, lengths, kv, d, t, held, page, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.page, self.held = rows, lengths, page, held
        self.kv, self.d, self.dtype = kv, d, TYPES[t]
        per = [(n + page - 1) // page for n in lengths]
        order = torch.randperm(sum(per) + 2, generator=g).tolist()
        width, at = max(per + [1]), 0
        table = []
        for n in per:
            table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.pages = ints(table).view(len(lengths), width)
        self.starts, self.lengths = starts_of(rows), ints(lengths)
        self.slots = len(order) * page
        free = torch.ones(self.slots, dtype=torch.bool)
        for i, n in enumerate(lengths):
            free[self.at(i, 0, n).cpu()] = False
        self.free = free.cuda()
        self.states, self.scales = [], []
        for _ in "kv":
            x = torch.randn(self.slots, kv, d, generator=g) * spread
            if held == "i8":
                top = x.abs().amax(-1, keepdim=True)
                self.states.append(torch.round(x * (127 / top)).to(torch.int8).cuda())
                s = (top[..., 0] / 127).cuda()
                s[self.free] = float("nan")
                self.scales.append(s)
            else:
                x = x.to(self.dtype).cuda()
                x[self.free] = float("nan")
                self.states.append(x)
                self.scales.append(None)

    def at(self, i, first, last):
        """The slots of sequence i's positions first .. last - 1."""
        p = torch.arange(first, last, device=self.pages.device)
        return self.pages[i].long()[p // self.page] * self.page + p % self.page

    def new_slots(self):
        return torch.cat([self.at(i, n - m, n) for i, (m, n) in enumerate(zip(self.rows, self.lens))])

    def values(self, which, slots):
        """What slots hold, in 64 bits."""
        x = self.states[which][slots].double()
        return x if self.held != "i8" else x * self.scales[which][slots].double()[..., None]

    def operand(self, T):
        return T.StateCache(self.states[0], self.states[1], self.page, *self.scales)

    def arrays(self):
        return self.starts, self.lengths, self.pages


def check_rows(out, q, first, k, v, window=0, scale=None, coded=None):
    """out, the attention of q's rows at positions first .. to the states k and v [n, kv, d] (64 bits), is the formula's.

    Tolerance, from the roundings that the operators state. A score is a sum of d F32 products in some order, times one
    or two factors and less a maximum: off by at most e = (d + 6) 2^-24 A + 2^-22 S, A the largest sum of |q_c k_c| scale
    and S the largest |score| of the row. A probability is then off by a factor of 1 +- (2 e + 2^-21) against its row's
    sum, by half a step of the type where it is rounded to it (16-bit operands), and, in F16, by half a step of the
    smallest number, 2^-25 of the row's largest. Times the scale of an I8 value (`coded`: the scales of v) that is what is
    rounded, in F16 against the largest scale: half a step is up to 2^-25 of the row's largest and 4 times the largest
    scale, for each code. The products with V are summed in F32 in some order, n 2^-24 each, and the output is rounded
    once."""
    m, heads, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    if m == 0:
        return
    scale = d ** -0.5 if scale is None else scale
    half, tiny = torch.finfo(out.dtype).eps / 2, torch.finfo(out.dtype).tiny
    f32 = out.dtype == torch.float32
    ks, vs = (x.repeat_interleave(heads // kv, 1) for x in (k, v))
    at = first + torch.arange(m, device="cuda")
    p = torch.arange(n, device="cuda")
    live = p[None] <= at[:, None]
    if window:
        live &= p[None] > at[:, None] - window
    qs, o = q.double(), out.double()
    none = ~live.any(1)
    assert (o[none] == 0).all()
    if none.all():
        return
    # (States that no row sees may hold anything.)
    seen = live.any(0)
    ks, vs = torch.where(seen[:, None, None], ks, 0.0), torch.where(seen[:, None, None], vs, 0.0)
    s = (torch.matmul(qs.transpose(0, 1), ks.permute(1, 2, 0)) * scale).masked_fill(~live, -float("inf"))
    pr = torch.softmax(s, -1).nan_to_num(0.0)
    want = torch.matmul(pr, vs.transpose(0, 1)).transpose(0, 1)
    a = torch.matmul(qs.abs().transpose(0, 1), ks.abs().permute(1, 2, 0)).masked_fill(~live, 0).amax(-1, keepdim=True)
    big = s.abs().masked_fill(~live, 0).amax(-1, keepdim=True)
    e = (d + 6) * 2.0 ** -24 * a * abs(scale) + 2.0 ** -22 * big
    off = 2 * e + 2.0 ** -21 + n * 2.0 ** -23 + (0 if f32 else half)
    weight = torch.matmul(pr * off, vs.abs().transpose(0, 1)).transpose(0, 1)
    if out.dtype == torch.float16:
        each = vs.abs()
        if coded is not None:
            cs = torch.where(seen[:, None], coded.double(), 0.0).repeat_interleave(heads // kv, 1)
            each = (vs / torch.where(cs > 0, cs, 1.0)[..., None]).abs() * 4 * cs.amax(0)[None, :, None]
        weight = weight + 2.0 ** -25 * (pr.amax(-1).transpose(0, 1)[..., None] * each.sum(0)[None])
    tol = weight * 1.01 + want.abs().clamp_min(tiny) * half * 1.01
    o, want, tol = o[~none], want[~none], tol[~none]
    assert torch.isfinite(o).all()
    worst = ((o - want).abs() / tol).max().item()
    assert worst <= 1, (m, n, worst)


def check(cache, q, out, window=0, scale=None):
    """out is the attention of q's rows over the cache's states."""
    row = 0
    for i, (m, n) in enumerate(zip(cache.rows, cache.lens)):
        at = cache.at(i, 0, n)
        coded = cache.scales[1][at] if cache.held == "i8" else None
        check_rows(out[row:row + m], q[row:row + m], n - m, cache.values(0, at), cache.values(1, at), window, scale, coded)
        row += m
