"""The decode operators' benchmark cases: appending to a paged 8-bit key/value cache with the
rotation of positions, attention over that cache, and products with 4-bit weights.

``run`` computes each operator in elementary torch operations (32 bits inside, rounded once at
the end) where ``own`` is false, and calls ``piton_b200.decode`` where it is true.  The cache
holds e4m3 codes ``[pages, kv_heads, page, dim]`` and one power-of-two scale per page and head;
4-bit weights are two per byte along the inner dimension with a scale (and optionally a zero
point) per group.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3_MAX = 448.0


def listed():
    return [
        # one token of one sequence of a small character model: the call's latency
        dict(name="append one token", op="append", batch=1, new=1, ragged=False, heads=4, kv_heads=4, dim=32, page=16,
             start=100, rot=32, interleaved=False, dtype="fp32"),
        # one token for each of 256 running sequences, grouped heads
        dict(name="append batch 256", op="append", batch=256, new=1, ragged=False, heads=32, kv_heads=8, dim=128, page=64,
             start=4000, rot=128, interleaved=False, dtype="bf16"),
        # prompts of different lengths appended together, a head per key head, half of each head rotated in pairs
        dict(name="append ragged prompts", op="append", batch=7, new=1500, ragged=True, heads=32, kv_heads=32, dim=64,
             page=32, start=333, rot=32, interleaved=True, dtype="fp32"),
        # four long prompts
        dict(name="append long prompts", op="append", batch=4, new=8192, ragged=False, heads=32, kv_heads=8, dim=128,
             page=64, start=0, rot=128, interleaved=False, dtype="bf16"),
        # one sequence of a small character model, within its 128 positions
        dict(name="attention short", op="attention", batch=1, new=1, length=100, ragged=False, heads=4, kv_heads=4, dim=32,
             page=16, window=0, dtype="fp32"),
        # one sequence with a long context: the keys are the only axis to split
        dict(name="attention long context", op="attention", batch=1, new=1, length=131000, ragged=False, heads=32,
             kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # a batch of sequences of different lengths, four tokens each checked at once, sliding window
        dict(name="attention window, 4 new", op="attention", batch=24, new=4, length=7001, ragged=True, heads=20, kv_heads=5,
             dim=128, page=32, window=2048, dtype="fp16"),
        # the benchmark's attention heads (32 of 64, 4096 positions) as a decode batch in 32 bits
        dict(name="attention batch 32 fp32", op="attention", batch=32, new=1, length=4096, ragged=False, heads=32,
             kv_heads=32, dim=64, page=64, window=0, dtype="fp32"),
        # the small character model's joint projection of queries, keys and values, one token
        dict(name="matvec 128 x 384", op="matvec", rows=1, inner=128, outer=384, group=32, zeros=False, bias=True,
             dtype="fp32"),
        # one token through a square layer
        dict(name="matvec 4096 x 4096", op="matvec", rows=1, inner=4096, outer=4096, group=128, zeros=False, bias=False,
             dtype="bf16"),
        # five tokens in 32 bits with zero points, sizes that no tile divides
        dict(name="matvec 8200 x 8191, 5 rows", op="matvec", rows=5, inner=8200, outer=8191, group=64, zeros=True, bias=True,
             dtype="fp32"),
        # sixteen tokens through a wide layer
        dict(name="matvec 8192 x 32768, 16 rows", op="matvec", rows=16, inner=8192, outer=32768, group=128, zeros=True,
             bias=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "matvec"))
    if op == "matvec":
        inner, outer = 8 * _log(rng, 4, 2048) + rng.choice((0, 0, 0, 2, 5)), _log(rng, 17, 33000)
        while inner * outer > 8192 * 32768:
            outer //= 2
        return dict(op=op, rows=_log(rng, 1, 16), inner=inner, outer=outer, group=rng.choice((32, 64, 128)),
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.5, dtype=rng.choice(("fp32", "bf16", "fp16")))
    kv_heads, group = rng.choice((1, 2, 4, 5, 8, 16, 32)), rng.choice((1, 1, 2, 3, 4, 8))
    dim = rng.choice((32, 64, 128))
    case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128)),
                dtype=rng.choice(("fp32", "bf16", "fp16")), ragged=rng.random() < 0.5, batch=_log(rng, 1, 256))
    if op == "append":
        case.update(new=_log(rng, 1, 8192) if rng.random() < 0.6 else 1, start=rng.randrange(0, 5000),
                    rot=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.5)
        most, key = 32768 * (32 + 16) * 128 * 2, "new"
        while case["batch"] * case["new"] * (case["heads"] + 2 * kv_heads) * dim * SIZE[case["dtype"]] > most:
            case["batch" if case["batch"] > 1 else key] //= 2
        return case
    case.update(new=rng.choice((1, 1, 1, 2, 4, 7)), length=_log(rng, 8, 131000),
                window=rng.choice((0, 0, 0, 128, 1000)))
    while case["batch"] * case["length"] * kv_heads * dim > 32 * 4096 * 32 * 64:
        case["batch" if case["batch"] > 1 else "length"] //= 2
    return case


def _news(case):
    """New tokens of each sequence."""
    n, b = case["new"], case["batch"]
    return [1 + (i * 7919 + 555) % (2 * n - 1) if case["ragged"] else n for i in range(b)]


def _lengths(case):
    """Tokens in the cache of each sequence: `start` or `length` at most, ragged ones down to half of it."""
    most = case["start"] if case["op"] == "append" else case["length"]
    spread = case["ragged"] or case["op"] == "append"
    return [max(0, most - (i * 40503) % (most // 2 + 1)) if spread else most for i in range(case["batch"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(case, pages, gen, used):
    """Codes whose blocks reach the type's largest values, scales around 2^-7; pages no table names stay zero."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = []
    for _ in range(2):
        codes = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        for lo in range(0, used.numel(), 4096):
            part = used[lo:lo + 4096]
            x = torch.randn((part.numel(),) + shape[1:], generator=gen, device="cuda") * 100.0
            codes[part] = x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        out.append(codes.view(torch.float8_e4m3fn))
    scales = [torch.ldexp(torch.ones(shape[:2], device="cuda"),
                          torch.randint(-8, -5, shape[:2], generator=gen, device="cuda")) for _ in range(2)]
    return out[0], out[1], scales[0], scales[1]


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "matvec":
        m, k, n, g = case["rows"], case["inner"], case["outer"], case["group"]
        groups, t = -(-k // g), DTYPES[case["dtype"]]
        return {"case": case,
                "x": torch.randn((m, k), generator=gen, device="cuda").to(t),
                "codes": torch.randint(0, 256, (n, -(-k // 2)), generator=gen, device="cuda", dtype=torch.uint8),
                "scales": ((0.5 + torch.rand((n, groups), generator=gen, device="cuda")) / (5.0 * math.sqrt(k))).to(t),
                "zeros": torch.randint(4, 12, (n, groups), generator=gen, device="cuda", dtype=torch.uint8)
                if case["zeros"] else None,
                "bias": torch.randn(n, generator=gen, device="cuda").to(t) if case["bias"] else None}
    b, page, t = case["batch"], case["page"], DTYPES[case["dtype"]]
    held, new = _lengths(case), _news(case) if case["op"] == "append" else [case["new"]] * b
    total = [h + n for h, n in zip(held, new)] if case["op"] == "append" else held
    need = [-(-x // page) for x in total]
    width, pages = max(1, max(need)), sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[at] = order[:sum(need)]
    state = {"case": case, "table": table}
    tokens = sum(new)
    shape = (tokens, case["heads"] + 2 * case["kv_heads"], case["dim"])
    if case["op"] == "attention":
        state["cache"] = _cache(case, pages, gen, table[at].long())
        state["q"] = torch.randn((tokens,) + (case["heads"], case["dim"]), generator=gen, device="cuda").to(t)
        state["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
        state["max_length"] = max(total)
        return state
    # only the pages that hold old tokens have contents
    old = torch.arange(width, device="cuda")[None, :] * page < torch.tensor(held, device="cuda")[:, None]
    state["cache"] = _cache(case, pages, gen, table[old].long())
    qkv = torch.randn(shape, generator=gen, device="cuda").to(t)     # one projection's output, split by views
    state["q"], state["k"], state["v"] = qkv.split((case["heads"], case["kv_heads"], case["kv_heads"]), dim=1)
    state["starts"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    state["cu"] = None
    if case["ragged"]:
        state["cu"] = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    r = case["rot"]
    angle = torch.arange(max(total), dtype=torch.float64, device="cuda")[:, None] * \
        10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def run(state):
    case = state["case"]
    if own:
        from piton_b200 import decode
        if case["op"] == "matvec":
            return decode.matvec_w4(state["x"], state["codes"], state["scales"], group=case["group"], zeros=state["zeros"],
                                    bias=state["bias"])
        if case["op"] == "attention":
            return decode.kv_attention(state["q"], state["cache"], state["table"], state["lengths"],
                                       window=case["window"], max_length=state["max_length"])
        q, lengths = decode.kv_append(state["k"], state["v"], state["cache"], state["table"], state["starts"],
                                      cu=state["cu"], q=state["q"], cos=state["cos"], sin=state["sin"],
                                      interleaved=case["interleaved"])
        return {"q": q, "lengths": lengths, "cache": state["cache"]}
    return {"append": _append, "attention": _attention, "matvec": _matvec}[case["op"]](state)


# ---- plain forms -----------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    c, s = cos[:, None], sin[:, None]
    y1, y2 = a * c - b * s, b * c + a * s
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., r:]), -1)


def _block_scale(a):
    """The least power of two s with a <= 448 s, between 2^-120 and 2^120."""
    m, e = torch.frexp(a)
    e = torch.where(a > 0, e - torch.where(m > 0.875, 8, 9), -120).clamp(-120, 120)
    return torch.ldexp(torch.ones_like(a), e)


def _append(state):
    case, table, starts = state["case"], state["table"].long(), state["starts"].long()
    page, width, b = case["page"], state["table"].shape[1], case["batch"]
    tokens = state["k"].shape[0]
    if state["cu"] is None:
        n = torch.full_like(starts, case["new"])
    else:
        n = (state["cu"][1:] - state["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), n, output_size=tokens)
    pos = starts[seq] + torch.arange(tokens, device="cuda") - (n.cumsum(0) - n)[seq]
    cos, sin = state["cos"][pos], state["sin"][pos]
    unit, slot = seq * width + pos // page, pos % page          # the page of a sequence, the token's place in it
    page_of = table.reshape(-1)
    first, held = (starts // page).clamp(max=width - 1), starts % page      # only a sequence's first page holds old tokens
    first_page = table.gather(1, first[:, None])[:, 0].clamp(min=0)
    keep = torch.arange(page, device="cuda") < torch.where(n > 0, held, 0)[:, None]
    k = _rotate(state["k"].float(), cos, sin, case["interleaved"])
    for x, codes, scales in ((k, state["cache"][0], state["cache"][2]), (state["v"].float(), state["cache"][1], state["cache"][3])):
        finite = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        units = torch.zeros((b * width, case["kv_heads"]), device="cuda")
        units.scatter_reduce_(0, unit[:, None].expand_as(finite), finite, "amax")
        before = torch.zeros_like(units)
        at = torch.arange(b, device="cuda") * width + first
        before[at] = torch.where((held > 0)[:, None], scales[first_page], 0.0)
        s = torch.maximum(_block_scale(units), before)
        old = codes[first_page].float()
        again = (old * (before[at] / s[at])[..., None, None]).to(codes.dtype)
        raw = codes.view(torch.uint8)
        raw[first_page] = torch.where(keep[:, None, :, None], again.view(torch.uint8), raw[first_page])
        y = torch.where(x.isfinite(), x / s[unit][..., None], math.nan)
        raw[page_of[unit], :, slot] = y.to(codes.dtype).view(torch.uint8)
        scales[page_of[unit]] = s[unit]
    q = _rotate(state["q"].float(), cos, sin, case["interleaved"]).to(state["q"].dtype)
    return {"q": q, "lengths": (starts + n).to(torch.int32), "cache": state["cache"]}


def _attention(state):
    case, (kc, vc, ks, vs) = state["case"], state["cache"]
    b, n, h, kvh, d, page = (case[x] for x in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    table = state["table"].long().clamp(min=0)
    keys = table.shape[1] * page
    k = (kc.view(torch.uint8)[table].view(kc.dtype).float() * ks[table][..., None, None]).transpose(2, 3).reshape(b, keys, kvh, d)
    v = (vc.view(torch.uint8)[table].view(vc.dtype).float() * vs[table][..., None, None]).transpose(2, 3).reshape(b, keys, kvh, d)
    q = state["q"].float().reshape(b, n, kvh, h // kvh, d)
    s = torch.einsum("bnhgd,bkhd->bhgnk", q, k) * (1.0 / math.sqrt(d))
    pos = state["lengths"].long()[:, None] - n + torch.arange(n, device="cuda")
    at = torch.arange(keys, device="cuda")
    seen = at <= pos[..., None]
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.einsum("bhgnk,bkhd->bnhgd", p, v)
    total = p.sum(-1).permute(0, 3, 1, 2)[..., None]
    o = torch.where(total > 0, o / total.clamp(min=1e-37), 0.0)
    return o.reshape(b * n, h, d).to(state["q"].dtype)


def _matvec(state):
    case, codes = state["case"], state["codes"]
    w = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :case["inner"]].float()
    group = torch.arange(case["inner"], device="cuda") // case["group"]
    zeros = state["zeros"].float()[:, group] if state["zeros"] is not None else 8.0
    w = (w - zeros) * state["scales"].float()[:, group]
    y = state["x"].float() @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


# ---- work and 64-bit values ----------------------------------------------------------------

def work(case):
    if case["op"] == "matvec":
        m, k, n, size = case["rows"], case["inner"], case["outer"], SIZE[case["dtype"]]
        groups = -(-k // case["group"])
        return {"bytes": n * -(-k // 2) + n * groups * (size + (1 if case["zeros"] else 0)) + m * (k + n) * size +
                (n * size if case["bias"] else 0), "flops": 2 * m * n * k}
    h, kvh, d, page, size = case["heads"], case["kv_heads"], case["dim"], case["page"], SIZE[case["dtype"]]
    held = _lengths(case)
    if case["op"] == "append":
        new = _news(case)
        tokens = sum(new)
        units = sum((s + n - 1) // page - s // page + 1 for s, n in zip(held, new))
        rows = min(tokens, max(s + n for s, n in zip(held, new)))
        return {"bytes": tokens * ((2 * h + 2 * kvh) * d * size + 2 * kvh * d) + units * (8 * kvh + 4) + rows * case["rot"] * 4 +
                8 * case["batch"], "flops": tokens * (3 * (h + kvh) * case["rot"] + 4 * kvh * d)}
    nbytes, flops = 0, 0
    for length in held:
        first = max(0, length - case["new"] + 1 - case["window"]) if case["window"] else 0
        nbytes += (length - first) * kvh * 2 * d + -(-length // page) * (4 + 8 * kvh)
        for i in range(case["new"]):
            pos = length - case["new"] + i
            seen = max(0, min(pos + 1, case["window"]) if case["window"] else pos + 1)
            flops += 4 * h * d * seen
    return {"bytes": nbytes + 2 * case["batch"] * case["new"] * h * d * size, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "matvec":
        n, k, g = case["outer"], case["inner"], case["group"]
        y = torch.empty((case["rows"], n), dtype=torch.float64, device="cuda")
        x = state["x"].double()
        step = max(1, (1 << 28) // k)
        for lo in range(0, n, step):
            c = state["codes"][lo:lo + step]
            w = torch.empty((c.shape[0], 2 * c.shape[1]), dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = c % 16, torch.div(c, 16, rounding_mode="floor")
            z = state["zeros"][lo:lo + step].double() if case["zeros"] else torch.full((c.shape[0], -(-k // g)), 8.0, dtype=torch.float64, device="cuda")
            s = state["scales"][lo:lo + step].double()
            w = (w[:, :k] - z.repeat_interleave(g, 1)[:, :k]) * s.repeat_interleave(g, 1)[:, :k]
            y[:, lo:lo + step] = x @ w.T
        return y + state["bias"].double() if case["bias"] else y
    return _exact_attention(case, state) if case["op"] == "attention" else _exact_append(case, state)


def _exact_attention(case, state):
    kc, vc, ks, vs = state["cache"]
    n, h, kvh, d, page = (case[x] for x in ("new", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros((case["batch"], n, kvh, h // kvh, d), dtype=torch.float64, device="cuda")
    q = state["q"].double().reshape(out.shape) / math.sqrt(d)
    for i, length in enumerate(_lengths(case)):
        ids = state["table"][i, :-(-length // page)].long()
        if not length:
            continue
        for j in range(kvh):
            k = (kc.view(torch.uint8)[ids, j].view(kc.dtype).double() * ks[ids, j].double()[:, None, None]).reshape(-1, d)[:length]
            v = (vc.view(torch.uint8)[ids, j].view(vc.dtype).double() * vs[ids, j].double()[:, None, None]).reshape(-1, d)[:length]
            for t in range(n):
                end = length - n + t + 1
                first = max(0, end - case["window"]) if case["window"] else 0
                if end > first:
                    out[i, t, j] = torch.softmax(q[i, t, j] @ k[first:end].T, -1) @ v[first:end]
    return out.reshape(-1, h, d)


def _e4m3(x):
    """The nearest e4m3 value, ties to the even one."""
    e = torch.frexp(x)[1].clamp(min=-5) - 1                      # 2^e <= |x| < 2^(e + 1); below 2^-6 the step is 2^-9
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return torch.round(x / step) * step


def _exact_append(case, state):
    kc, vc, ks, vs = state["cache"]
    out = [kc.double(), vc.double(), ks.double(), vs.double()]
    page, r = case["page"], case["rot"]
    new, held = _news(case), _lengths(case)
    if sum(new) > 40000 or sum(-(-n // page) + 1 for n in new) > 6000:
        return None
    if case["interleaved"]:
        first = torch.arange(0, r, 2, device="cuda")
        second = first + 1
    else:
        first = torch.arange(r // 2, device="cuda")
        second = first + r // 2

    def rotated(x, lo):
        c, s = (state[w][lo:lo + x.shape[0]].double()[:, None] for w in ("cos", "sin"))
        y = x.double().clone()
        y[..., first] = x[..., first].double() * c - x[..., second].double() * s
        y[..., second] = x[..., second].double() * c + x[..., first].double() * s
        return y

    q = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, start) in enumerate(zip(new, held)):
        q[at:at + n] = rotated(state["q"][at:at + n], start)
        values = rotated(state["k"][at:at + n], start), state["v"][at:at + n].double()
        at, done = at + n, 0
        while done < n:
            place, inside = divmod(start + done, page)
            count, at_page = min(n - done, page - inside), int(state["table"][i, place])
            for x, codes, scales in zip(values, out[:2], out[2:]):
                block = x[done:done + count].transpose(0, 1)
                a = block.abs().amax((1, 2))
                s = torch.exp2(torch.ceil(torch.log2(a / E4M3_MAX)).clamp(-120, 120))
                if inside:
                    before = scales[at_page].clone()
                    s = torch.maximum(s, before)
                    codes[at_page, :, :inside] = _e4m3(codes[at_page, :, :inside] * (before / s)[:, None, None])
                codes[at_page, :, inside:inside + count] = _e4m3(block / s[:, None, None])
                scales[at_page] = s
            done += count
    return {"q": q, "lengths": None, "cache": tuple(out)}
