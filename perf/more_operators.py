"""The operators of a program's own tokens, as they are timed: attention over a prompt, and over a cache of states.

A program that generates or reads step by step over a session's states keeps the keys and values of its tokens: it runs
the attention of a whole prompt (causal, packed sequences), writes the prompt's keys and values into the pages of a
cache (as they are, or as int8 codes), attends with each next token or chunk of tokens over the cache, and reads states
back out of it.

The widths are those of the encoders in turboembed_amd/workloads.py (12 and 16 heads of 64) and generic ones beside them
(shared key heads, heads of 80 and 128). Lengths are spread evenly over [lo, hi], so every seed has the same work.
"""
import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _prompt(name, t, seqs, lo, hi, heads, kv, d, window=0):
    c = dict(op="prompt", t=t, seqs=seqs, mlo=lo, mhi=hi, llo=lo, lhi=hi, heads=heads, kv=kv, d=d, window=window)
    return dict(c, name=name) if name else c


def _cached(op, name, t, held, seqs, mlo, mhi, llo, lhi, heads, kv, d, page, window=0):
    """seqs sequences of mlo to mhi new tokens, after which llo to lhi states are in pages of `page`, as t or i8."""
    c = dict(op=op, t=t, held=held, seqs=seqs, mlo=mlo, mhi=mhi, llo=llo, lhi=lhi, heads=heads, kv=kv, d=d, page=page,
             window=window)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One short question: a launch and its latency.
        _prompt("prompt-query-f16", "f16", 1, 23, 23, 12, 12, 64),
        # A batch of passages in the exact tier.
        _prompt("prompt-passages-f32", "f32", 24, 20, 500, 12, 12, 64),
        # Long documents, four heads to a key head.
        _prompt("prompt-bulk-bf16", "bf16", 8, 2048, 8192, 32, 8, 128),
        # One token of one sequence: a short time on a whole card.
        _cached("attend", "step-one-bf16", "bf16", "bf16", 1, 1, 1, 4096, 4096, 16, 4, 64, 16),
        # One token each of a serving batch, contexts of every length.
        _cached("attend", "step-batch-bf16", "bf16", "bf16", 64, 1, 1, 200, 8192, 32, 8, 128, 16),
        # The same with int8 states, every head its own.
        _cached("attend", "step-batch-i8-f16", "f16", "i8", 96, 1, 1, 100, 6000, 12, 12, 64, 64),
        # Chunks of long prompts over the int8 states before them.
        _cached("attend", "chunk-i8-bf16", "bf16", "i8", 8, 512, 512, 1024, 8192, 32, 8, 128, 32),
        # Uneven chunks in the exact tier, pages that no tile divides, a sliding window.
        _cached("attend", "chunk-odd-f32", "f32", "f32", 11, 3, 61, 61, 1900, 6, 2, 80, 24, 700),
        # A step's tokens into their pages.
        _cached("write", "write-step-f16", "f16", "f16", 48, 1, 1, 100, 600, 16, 16, 64, 16),
        # Whole prompts into int8 pages.
        _cached("write", "write-bulk-i8-bf16", "bf16", "i8", 8, 4096, 4096, 4096, 4096, 8, 8, 128, 64),
        # A few short prefixes of an odd width.
        _cached("read", "read-odd-bf16", "bf16", "bf16", 9, 1, 333, 1, 400, 3, 3, 80, 24),
        # Cached documents back as 16-bit rows.
        _cached("read", "read-bulk-i8-f16", "f16", "i8", 8, 2048, 4096, 2048, 4096, 16, 16, 64, 32),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """One more case: any operator, its sizes log-uniform from one token up."""
    op = rng.choice(["prompt", "prompt", "attend", "attend", "attend", "write", "read"])
    t = rng.choice(["f16", "bf16", "bf16", "f32"])
    d = rng.choice([32, 64, 64, 80, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 2, 4, 8] if kv <= 4 else [1, 1, 4])
    window = _log(rng, 16, 4096) if rng.random() < 0.25 else 0
    # (At most a quarter of the largest listed case's scores; F32's products have a sixteenth of the rate.)
    scores = (1 << 30) >> (4 if t == "f32" else 0)
    if op == "prompt":
        hi = _log(rng, 4, 8192)
        while hi > 64 and heads * hi * hi > 2 * scores:
            hi = hi * 3 // 4
        seqs = _log(rng, 1, max(1, min(64, 2 * scores // (heads * hi * hi))))
        return _prompt("", t, seqs, max(1, int(hi * rng.choice([0.1, 0.5, 1.0]))), hi, heads, kv, d, window)
    held = rng.choice([t, "i8"])
    page = rng.choice([16, 16, 24, 32, 64, 128])
    if op == "attend":
        lhi = _log(rng, 16, 16384)
        mhi = 1 if rng.random() < 0.5 else min(lhi, _log(rng, 2, 1024))
        seqs = _log(rng, 1, max(1, min(128, scores // (heads * mhi * lhi), (1 << 28) // (kv * d * lhi))))
    else:
        mhi = _log(rng, 1, 4096)
        seqs = _log(rng, 1, max(1, min(64, (1 << 25) // (kv * d * mhi))))
        lhi, window = mhi + rng.choice([0, 37, 300]), 0
    mlo = max(1, int(mhi * rng.choice([0.1, 1.0])))
    return _cached(op, "", t, held, seqs, mlo, mhi, max(mlo, int(lhi * rng.choice([0.1, 0.6]))), lhi, heads, kv, d, page,
                   window)


# ---- what a program has in hand before the call -------------------------------------

def _spread(seqs, lo, hi):
    return [hi if seqs == 1 else lo + (hi - lo) * i // (seqs - 1) for i in range(seqs)]


def _lengths(c):
    """(new tokens, states) of each sequence."""
    new = _spread(c["seqs"], c["mlo"], c["mhi"])
    return new, [max(m, n) for m, n in zip(new, _spread(c["seqs"], c["llo"], c["lhi"]))]


@functools.lru_cache(maxsize=None)
def _context():
    import turboembed_amd as T
    return T.Runtime().context(0)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _coded(x):
    """int8 codes of rows and their scales."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127 / top.clamp_min(1e-30))).to(torch.int8), top[..., 0] / 127


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"op": case["op"], "case": case}
    if own:
        s["ctx"] = _context()
    new, held = _lengths(c)
    t, heads, kv, d, tokens = TYPES[c["t"]], c["heads"], c["kv"], c["d"], sum(new)
    s["new"], s["held"] = new, held
    firsts = [0]
    for m in new:
        firsts.append(firsts[-1] + m)
    s["starts"] = _ints(firsts)

    def rows(n, *heads_and_width):
        """Projections: tokens of different size, a few columns of each head larger than the rest."""
        x = torch.randn(n, *heads_and_width, generator=g, device="cuda")
        x *= torch.exp(0.3 * torch.randn(n, *[1] * len(heads_and_width), generator=g, device="cuda"))
        return x * torch.where(torch.rand(heads_and_width, generator=g, device="cuda") < 0.02, 3.0, 1.0)

    if c["op"] in ("prompt", "attend"):
        s["q"] = rows(tokens, heads, d).to(t)
        s["out"] = torch.empty(tokens, heads, d, dtype=t, device="cuda")
    if c["op"] == "prompt":
        # Keys and values side by side, as one product writes them.
        both = rows(tokens, 2, kv, d).to(t)
        s["k"], s["v"] = both[:, 0], both[:, 1]
        return s
    # Pages in no order, a few of them nobody's.
    page, per = c["page"], [(n + c["page"] - 1) // c["page"] for n in held]
    order = torch.randperm(sum(per) + 5, generator=g, device="cuda").to(torch.int32)
    s["pages"] = torch.zeros(len(held), max(per), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        s["pages"][i, :n] = order[at:at + n]
        at += n
    s["lengths"] = _ints(held)
    slots = (sum(per) + 5) * page
    for name in ("k", "v"):
        x = rows(slots, kv, d)
        if c["held"] == "i8":
            s["c" + name], s["s" + name] = _coded(x)
        else:
            s["c" + name], s["s" + name] = x.to(t), None
    if c["op"] == "write":
        both = rows(tokens, 2, kv, d).to(t)
        s["k"], s["v"] = both[:, 0], both[:, 1]
        # (Where a program wants the values of int8 states: the rows' type.)
        s["values"] = [torch.empty(slots, kv, d, dtype=t, device="cuda") for _ in "kv"] if c["held"] == "i8" else None
    if c["op"] == "read":
        s["k"], s["v"] = (torch.empty(tokens, kv, d, dtype=t, device="cuda") for _ in "kv")
    if c["op"] == "attend":
        # What stands in slots that hold no state is nobody's value.
        free = torch.ones(slots, dtype=torch.bool, device="cuda")
        free[_slots(s, [0] * len(held), held)] = False
        for name in ("sk", "sv") if c["held"] == "i8" else ("ck", "cv"):
            s[name][free] = float("nan")
    if own:
        import turboembed_amd as T
        s["cache"] = T.StateCache(s["ck"], s["cv"], page, k_scales=s["sk"], v_scales=s["sv"])
        if c["op"] == "attend":
            need = s["ctx"].cache_workspace(tokens, len(new), heads, kv, d, t)
            s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return s


def _slots(s, first, last):
    """The slots of positions first[i] .. last[i] - 1 of every sequence, one sequence after another."""
    page, found = s["case"]["page"], []
    for i, (a, b) in enumerate(zip(first, last)):
        p = torch.arange(a, b, device="cuda")
        found.append(s["pages"][i].long()[p // page] * page + p % page)
    return torch.cat(found)


# ---- one pass ---------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    if s["op"] == "prompt":
        return _plain_prompt(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    # The slot of each new token.
    page, row = s["case"]["page"], torch.arange(sum(s["new"]), device="cuda")
    i = torch.repeat_interleave(torch.arange(len(s["new"]), device="cuda"), s["starts"][1:] - s["starts"][:-1],
                                output_size=len(row))
    p = s["lengths"][i] - s["starts"][i + 1] + row
    at = s["pages"][i, p // page].long() * page + p % page
    if s["op"] == "read":
        return [_values(s, name, at).to(s["k"].dtype) for name in "kv"]
    return _plain_write(s, at)


def _own(s):
    ctx, stream, window = s["ctx"], torch.cuda.current_stream().cuda_stream, s["case"]["window"]
    if s["op"] == "prompt":
        ctx.prompt_attention(s["q"], s["k"], s["v"], s["starts"], s["out"], window=window, stream=stream)
        return s["out"]
    if s["op"] == "attend":
        ctx.cache_attention(s["q"], s["cache"], s["starts"], s["lengths"], s["pages"], s["out"], window=window,
                            workspace=s["workspace"], stream=stream)
        return s["out"]
    if s["op"] == "read":
        ctx.cache_read(s["cache"], s["starts"], s["lengths"], s["pages"], s["k"], s["v"], stream=stream)
        return [s["k"], s["v"]]
    ctx.cache_write(s["k"], s["v"], s["cache"], s["starts"], s["lengths"], s["pages"], stream=stream)
    return _held(s)


def _held(s):
    """The whole cache after a write: the states, or the values that codes stand for and the scales."""
    if s["sk"] is None:
        return [s["ck"], s["cv"]]
    values = [torch.mul(s["c" + name], s["s" + name][..., None], out=out) for name, out in zip("kv", s["values"])]
    return values + [s["sk"], s["sv"]]


def _values(s, name, at):
    x = s["c" + name][at].float()
    return x if s["sk"] is None else x * s["s" + name][at][..., None]


def _plain_write(s, at):
    for name in "kv":
        x = s[name]
        if s["sk"] is not None:
            # (64 bits: a value next to the border of two codes.)
            x = x.double()
            top = x.abs().amax(-1)
            s["s" + name][at] = (top / 127).float()
            x = torch.round(127 * x / torch.where(top > 0, top, 1.0)[..., None]).to(torch.int8)
        s["c" + name][at] = x
    return _held(s)


def _weights(p, live):
    """Softmax over the last axis of scores p in place, over the live ones (a row of none: zeros)."""
    p.masked_fill_(~live, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, 1.0, total))


def _plain_prompt(s):
    c, outs, at = s["case"], [], 0
    for m in s["new"]:
        q, k, v = (s[name][at:at + m].float() for name in "qkv")
        at += m
        # Heads that share a key head are rows of one product.
        q = q.view(m, c["kv"], -1, c["d"]).permute(1, 2, 0, 3).flatten(1, 2).contiguous()
        p = torch.matmul(q, k.permute(1, 2, 0).contiguous()).mul_(1 / math.sqrt(c["d"])).unflatten(1, (-1, m))
        i = torch.arange(m, device="cuda")
        live = i[None] <= i[:, None]
        if c["window"]:
            live &= i[None] > i[:, None] - c["window"]
        o = torch.matmul(_weights(p, live).flatten(1, 2), v.transpose(0, 1).contiguous()).unflatten(1, (-1, m))
        outs.append(o.permute(2, 0, 1, 3).flatten(1, 2))
    return torch.cat(outs).to(s["out"].dtype)


def _plain_attend(s):
    c, n, most, longest = s["case"], len(s["new"]), max(s["new"]), max(s["held"])
    kv, d, share, page = c["kv"], c["d"], c["heads"] // c["kv"], c["page"]
    new, held = (s["starts"][1:] - s["starts"][:-1])[:, None], s["lengths"][:, None]
    # A padded layout: row j and state p of every sequence.
    j, p = torch.arange(most, device="cuda"), torch.arange(longest, device="cuda")
    row = torch.where(j < new, s["starts"][:-1, None] + j, 0)
    slot = torch.where(p < held, s["pages"].long()[:, p // page] * page + p % page, 0)
    there = (p < held)[:, :, None, None]
    k, v = (torch.where(there, _values(s, name, slot), 0.0) for name in "kv")
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    q = s["q"].float()[row].view(n, most, kv, share, d).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()
    scores = torch.matmul(q, k).mul_(1 / math.sqrt(d)).unflatten(2, (share, most))
    at = (held - new + j)[:, :, None]
    live = (p <= at) & (p < held[:, :, None])
    if c["window"]:
        live &= p > at - c["window"]
    o = torch.matmul(_weights(scores, live[:, None, None]).flatten(2, 3), v).unflatten(2, (share, most))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[j < new].to(s["out"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------

def _pairs(m, n, window):
    """(pairs of m new tokens and the states that they see of n, the states that any of them sees)."""
    first = n - m
    if not window or window >= n:
        return m * first + m * (m + 1) // 2, n
    full = max(0, min(m, window - first))       # rows that see all before them
    pairs = full * first + full * (full + 1) // 2 + (m - full) * window
    return pairs, n - max(0, first + 1 - window)


def work(case):
    c = case
    new, held = _lengths(c)
    tokens, size, wide = sum(new), SIZE[c["t"]], c["kv"] * c["d"]
    seen = [_pairs(m, n, c["window"]) for m, n in zip(new, held)]
    if c["op"] in ("prompt", "attend"):
        state = 2 * wide * size if c.get("held") != "i8" else 2 * wide + 8 * c["kv"]
        return {"bytes": 2 * tokens * c["heads"] * c["d"] * size + sum(n for _, n in seen) * state,
                "flops": 4 * c["d"] * c["heads"] * sum(n for n, _ in seen)}
    state = 2 * wide + 8 * c["kv"] if c["held"] == "i8" else 2 * wide * size
    return {"bytes": tokens * (2 * wide * size + state), "flops": 4 * tokens * wide}


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    share = c["heads"] // c["kv"]

    def held(name, i, first, last):
        """Positions first .. last - 1 of sequence i as they stand in the cache."""
        where = [(p // c["page"], p % c["page"]) for p in range(first, last)]
        pages = s["pages"][i].tolist()
        at = torch.tensor([pages[a] * c["page"] + b for a, b in where], dtype=torch.long, device="cuda")
        x = s["c" + name].index_select(0, at).double()
        return x if c["held"] != "i8" else s["s" + name].index_select(0, at).double().unsqueeze(-1) * x

    if c["op"] == "write":
        want = []
        for name in "kv":
            values = s["c" + name].double()
            if c["held"] == "i8":
                values = values * s["s" + name].double().unsqueeze(-1)
            scales, row = None if c["held"] != "i8" else s["s" + name].double(), 0
            x = s[name].double()
            for i, (m, n) in enumerate(zip(s["new"], s["held"])):
                pages = s["pages"][i].tolist()
                at = torch.tensor([pages[p // c["page"]] * c["page"] + p % c["page"] for p in range(n - m, n)],
                                  dtype=torch.long, device="cuda")
                y = x[row:row + m]
                row += m
                if scales is not None:
                    step = torch.linalg.vector_norm(y, ord=math.inf, dim=2) / 127
                    unit = torch.where(step == 0, 1.0, step).unsqueeze(2)
                    y = torch.round(y / unit) * unit
                    scales.index_copy_(0, at, step)
                values.index_copy_(0, at, y)
            want.append((values, scales))
        return [w[0] for w in want] + ([] if c["held"] != "i8" else [w[1] for w in want])
    if c["op"] == "read":
        return [torch.cat([held(name, i, n - m, n) for i, (m, n) in enumerate(zip(s["new"], s["held"]))])
                for name in "kv"]
    out, row = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (m, n) in enumerate(zip(s["new"], s["held"])):
        if c["op"] == "prompt":
            k, v = s["k"][row:row + m].double(), s["v"][row:row + m].double()
        else:
            k, v = held("k", i, 0, n), held("v", i, 0, n)
        position = torch.arange(n - m, n, device="cuda")
        behind = position.unsqueeze(1) - torch.arange(n, device="cuda").unsqueeze(0)
        hidden = behind < 0 if not c["window"] else (behind < 0) | (behind >= c["window"])
        for h in range(c["heads"]):
            scores = torch.mm(s["q"][row:row + m, h].double(), k[:, h // share].t()) / math.sqrt(c["d"])
            out[row:row + m, h] = torch.mm(torch.softmax(scores.masked_fill_(hidden, -math.inf), 1), v[:, h // share])
        row += m
    return out
