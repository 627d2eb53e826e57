"""Performance cases of the operators a decode step makes around its experts: page plan, query and key preparation,
attention over the paged cache, and what is read off the output head's logits.

A case names one operator and its sizes.  `listed()` is the fixed set, `draw()` gives more of the same ranges.  64 query
heads and 16 key-value heads of 128 are what the FP8 projections [12288, 4096] and [4096, 8192] of this repository's
configurations belong to; 129280 is the vocabulary of its output head.

    plan      block tables, slots and positions of a step's new tokens (plan_pages)
    rope      norms of q and k per head, position rotation, cache write (qk_norm_rope)
    attend    one new token per request over the paged cache (paged_attention)
    logprobs  log probabilities, entropy and alternatives of sampled tokens (token_logprobs)

The plain forms below compute in float32 whatever the inputs' type (angles in float64) and round once at the end.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
MOST_CACHE = 131072 * 8 * 128 * 4  # bytes of keys and values of the largest attention case
MOST_PADDED = 64 * 8192 * 8 * 128  # elements of the keys padded to the longest request, as the plain form holds them


def _case(name, kind, **sizes):
    return {"name": name, "kind": kind, **sizes}


def listed():
    return [
        # one decode step of a serving batch: a token each, a page boundary now and then
        _case("plan-decode-64", "plan", requests=64, context=32768, tokens=64, page=16, mode="decode"),
        # a step that mixes decoding requests with prompt chunks, padded to its captured size
        _case("plan-mixed-256", "plan", requests=256, context=32768, tokens=16384, page=64, mode="mixed"),
        # a handful of concurrent sessions
        _case("rope-4", "rope", tokens=4, heads=64, kv_heads=16, dim=128, rotary=128, layout="half", yarn=False, norm=True, dtype="bf16", cache="bf16", page=64),
        # a full prompt chunk, half of every head rotated, long-context frequencies
        _case("rope-4096", "rope", tokens=4096, heads=64, kv_heads=16, dim=128, rotary=64, layout="half", yarn=True, norm=True, dtype="bf16", cache="bf16", page=64),
        # the ragged last chunk of a prompt into an FP8 cache
        _case("rope-fp8-777", "rope", tokens=777, heads=40, kv_heads=8, dim=96, rotary=96, layout="interleaved", yarn=False, norm=True, dtype="f16", cache="fp8", page=24),
        # a single session, short context
        _case("attend-1-1000", "attend", requests=1, longest=1000, spread="fixed", heads=64, kv_heads=16, dim=128, page=64, window=0, softcap=0.0, dtype="bf16", cache="bf16", lse=False),
        # a serving batch of very different lengths
        _case("attend-ragged-32", "attend", requests=32, longest=8192, spread="log", heads=64, kv_heads=16, dim=128, page=64, window=0, softcap=0.0, dtype="bf16", cache="bf16", lse=False),
        # a single session with a long document
        _case("attend-1-131072", "attend", requests=1, longest=131072, spread="fixed", heads=64, kv_heads=8, dim=128, page=64, window=0, softcap=0.0, dtype="bf16", cache="bf16", lse=True),
        # a full serving batch over an FP8 cache
        _case("attend-fp8-64", "attend", requests=64, longest=8192, spread="even", heads=64, kv_heads=8, dim=128, page=16, window=0, softcap=0.0, dtype="bf16", cache="fp8", lse=False),
        # layers with a sliding window and capped scores, small heads, an odd group, a page size that is no power of two
        _case("attend-window-48", "attend", requests=48, longest=16000, spread="even", heads=20, kv_heads=4, dim=64, page=24, window=1024, softcap=50.0, dtype="f16", cache="f16", lse=True),
        # a sampled token with its alternatives, logits as the head gives them
        _case("logprobs-1", "logprobs", rows=1, vocab=129280, dtype="f32", top=20, masked=0.0),
        # a scored prompt chunk
        _case("logprobs-512", "logprobs", rows=512, vocab=129280, dtype="bf16", top=8, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "attend", "attend", "attend", "logprobs"])
    c = {"kind": kind}
    if kind == "plan":
        c["mode"] = rng.choice(["decode", "mixed"])
        c["requests"] = _log_int(rng, 1, 256)
        c["context"] = _log_int(rng, 1, 32768)
        c["tokens"] = c["requests"] + rng.choice([0, rng.randint(1, 32)]) if c["mode"] == "decode" else _log_int(rng, 2 * c["requests"], 16384)
        c["page"] = rng.choice([8, 16, 24, 32, 64, 128])
        return c
    if kind == "logprobs":
        c["dtype"] = rng.choice(["f32", "bf16", "f16"])
        c["vocab"] = _log_int(rng, 1000, 200000)
        c["rows"] = _log_int(rng, 1, max(1, 512 * 129280 * 2 // (c["vocab"] * BYTES[c["dtype"]])))
        c["rows"] = min(c["rows"], 4096)
        c["top"] = rng.choice([0, 1, 5, 8, 20, 32])
        c["masked"] = rng.choice([0.0, 0.0, 0.9])  # share of the vocabulary that a grammar rules out
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    c["cache"] = rng.choice([c["dtype"], c["dtype"], "fp8"])
    c["dim"] = rng.choice([64, 96, 128, 128, 192, 256])
    c["kv_heads"] = rng.choice([1, 2, 4, 8, 16])
    c["heads"] = c["kv_heads"] * rng.randint(1, 64 // c["kv_heads"] if c["kv_heads"] > 2 else 24)
    c["page"] = rng.choice([8, 16, 24, 32, 64, 128])
    if kind == "rope":
        c["rotary"] = rng.choice([c["dim"], c["dim"] // 2, 2 * rng.randint(1, c["dim"] // 2)])
        c["layout"] = rng.choice(["half", "interleaved"])
        c["yarn"] = rng.choice([False, True])
        c["norm"] = rng.choice([True, True, False])
        most = 4096 * 96 * 128 // ((c["heads"] + 2 * c["kv_heads"]) * c["dim"])
        c["tokens"] = _log_int(rng, 1, min(most, 32768))
    else:
        c["requests"] = _log_int(rng, 1, 256)
        c["spread"] = rng.choice(["log", "even"]) if c["requests"] > 1 else "fixed"
        each = c["kv_heads"] * c["dim"]
        most = min(MOST_CACHE // (2 * BYTES[c["cache"]] * each * c["requests"]), MOST_PADDED // (each * c["requests"]), 131072)
        c["longest"] = _log_int(rng, min(16, most), most)
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        c["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
        c["lse"] = rng.choice([False, True])
    return c


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lens(c):
    """The lengths of a batch: the quantiles of their distribution, so that every seed has the same amount of work; in batches
    of 16 and more the last row is the padding of a captured batch."""
    n, most = c["requests"], c["longest"]
    if c["spread"] == "fixed":
        return [most] * n
    q = [(i + 0.5) / n for i in range(n)]
    lens = [max(1, round(most ** u if c["spread"] == "log" else u * most)) for u in q]
    return lens if n < 16 else lens[1:] + [0]


def _shuffled(lens, gen):
    x = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if len(lens) >= 16:
        return torch.cat([x[:-1][torch.randperm(len(lens) - 1, device=DEV, generator=gen)], x[-1:]])
    return x[torch.randperm(len(lens), device=DEV, generator=gen)]


def _tables(used, width, pages, gen):
    """Block tables of requests that hold `used` pages each, drawn from a pool, and the pages that are left."""
    perm = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((used.numel(), width), -1, dtype=torch.int32, device=DEV)
    mask = torch.arange(width, device=DEV)[None] < used[:, None]
    n = int(mask.sum())
    table[mask] = perm[:n]
    return table, perm[n:].contiguous()


def _values(shape, name, gen):
    """Keys or values as a cache holds them, with the scale of every head (None: none)."""
    if name != "fp8":
        return torch.randn(shape, device=DEV, generator=gen, dtype=DTYPES[name]), None
    scale = (torch.rand(shape[1], device=DEV, generator=gen) + 0.5) / 64
    x = torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16) * 64
    return x.to(torch.float8_e4m3fn), scale


def _frequencies(c):
    """Angle per position of every pair, in 64 bits on the host as a program sets them up once, and the size of the rotated vector."""
    r = c["rotary"]
    f = [10000.0 ** (-2.0 * i / r) for i in range(r // 2)]
    if not c["yarn"]:
        return torch.tensor(f, dtype=torch.float64, device=DEV), 1.0
    factor, trained = 32.0, 4096  # frequencies that turn less than once over the trained length are stretched, fast ones are kept
    at = lambda turns: r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
    keep = [1.0 - min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(r // 2)]
    f = [x * k + x / factor * (1.0 - k) for x, k in zip(f, keep)]
    return torch.tensor(f, dtype=torch.float64, device=DEV), 0.1 * math.log(factor) + 1.0


def prepare(c, seed):
    gen, s = _gen(seed), {"case": c}
    if c["kind"] == "plan":
        n, page = c["requests"], c["page"]
        ctx = torch.exp(torch.rand(n, device=DEV, generator=gen) * math.log(c["context"] + 1)).to(torch.int32) - 1
        if c["mode"] == "decode":  # one token each; a request in sixteen has just ended
            new = (torch.rand(n, device=DEV, generator=gen) > 1 / 16).to(torch.int32)
        else:  # half of the requests decode, the others share what is left of nine tenths of the step
            chunk = torch.rand(n, device=DEV, generator=gen) * (torch.rand(n, device=DEV, generator=gen) > 0.5)
            room = max(0, c["tokens"] * 9 // 10 - n)
            new = (chunk / chunk.sum().clamp_min(1e-6) * room).to(torch.int32) + 1
        used = (ctx + page - 1) // page
        width = (c["context"] + c["tokens"]) // page + 2
        pages = int(used.sum()) + n + c["tokens"] // page + 64
        s["ctx"], s["new"] = ctx, new
        s["table"], s["free"] = _tables(used, width, pages, gen)
        s["count"] = torch.tensor([s["free"].numel()], dtype=torch.int32, device=DEV)
    elif c["kind"] == "rope":
        t, h, g, d, page = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
        dt = DTYPES[c["dtype"]]
        s["qkv"] = torch.randn((t, (h + 2 * g) * d), device=DEV, generator=gen).mul_(1.5).to(dt)  # as the projection gives it
        for w in ("qw", "kw"):
            s[w] = (1 + 0.1 * torch.randn(d, device=DEV, generator=gen)).to(dt) if c["norm"] else None
        s["freq"], s["magnitude"] = _frequencies(c)
        first = torch.randint(0, 131072 if c["yarn"] else 16384, (1,), device=DEV, generator=gen, dtype=torch.int32)
        s["positions"] = first + torch.arange(t, device=DEV, dtype=torch.int32)
        pages = 2 * (t // page) + 8
        (s["kc"], s["ks"]), (s["vc"], s["vs"]) = (_values((pages, g, page, d), c["cache"], gen) for _ in "kv")
        perm = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
        step = first % page + torch.arange(t, device=DEV, dtype=torch.int32)
        s["slots"] = perm[(step // page).long()] * page + step % page
        if t >= 64:
            s["slots"][t - t // 64:] = -1  # padding of the step
    elif c["kind"] == "attend":
        page, lens = c["page"], _lens(c)
        s["lens"] = _shuffled(lens, gen)
        used = (s["lens"] + page - 1) // page
        pages = sum(-(-n // page) for n in lens) + 7
        s["table"], _ = _tables(used, -(-max(lens) // page), pages, gen)
        shape = (pages, c["kv_heads"], page, c["dim"])
        (s["kc"], s["ks"]), (s["vc"], s["vs"]) = (_values(shape, c["cache"], gen) for _ in "kv")
        s["q"] = torch.randn((c["requests"], c["heads"], c["dim"]), device=DEV, generator=gen).mul_(2).to(DTYPES[c["dtype"]])
    else:
        x = torch.randn((c["rows"], c["vocab"]), device=DEV, generator=gen).mul_(2.5)
        x.scatter_(1, torch.randint(0, c["vocab"], (c["rows"], 8), device=DEV, generator=gen), 11.0 + torch.rand((c["rows"], 8), device=DEV, generator=gen) * 4)
        s["tokens"] = torch.randint(0, c["vocab"], (c["rows"],), device=DEV, generator=gen, dtype=torch.int32)
        if c["masked"]:
            out = torch.rand((c["rows"], c["vocab"]), device=DEV, generator=gen) < c["masked"]
            out.scatter_(1, s["tokens"][:, None].long(), False)
            x.masked_fill_(out, -math.inf)
        s["logits"] = x.to(DTYPES[c["dtype"]])
    return s


def _heads(s):
    """q, k and v as views of the projection's rows."""
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].view(c["tokens"], h + 2 * g, d)
    return x[:, :h], x[:, h:h + g], x[:, h + g:]


# ---- one pass -------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"plan": _plain_plan, "rope": _plain_rope, "attend": _plain_attend, "logprobs": _plain_logprobs}[c["kind"]](s, c)


def _run_own(s, c):
    import cachalot_b200 as cb

    if c["kind"] == "plan":
        p = cb.plan_pages(s["ctx"], s["new"], s["table"], s["free"], s["count"], page_size=c["page"], tokens=c["tokens"])
        return {"starts": p.starts, "requests": p.requests, "positions": p.positions, "slots": p.slots, "lens": p.lens, "count": p.free_count, "table": s["table"]}
    if c["kind"] == "rope":
        q, k, v = _heads(s)
        y, _ = cb.qk_norm_rope(q, k, s["positions"], s["freq"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, interleaved=c["layout"] == "interleaved",
                               magnitude=s["magnitude"], v=v, k_cache=s["kc"], v_cache=s["vc"], slots=s["slots"], k_scale=s["ks"], v_scale=s["vs"])
        return {"q": y, "k": s["kc"], "v": s["vc"]}
    if c["kind"] == "attend":
        y = cb.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], window=c["window"], softcap=c["softcap"], k_scale=s["ks"], v_scale=s["vs"],
                               want_lse=c["lse"])
        return {"out": y[0], "lse": y[1]} if c["lse"] else {"out": y}
    r = cb.token_logprobs(s["logits"], s["tokens"], top=c["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    return {**out, "ids": r.top_ids, "top": r.top_logprobs} if c["top"] else out


def _plain_plan(s, c):
    page, tokens, table = c["page"], c["tokens"], s["table"]
    width = table.shape[1]
    ctx, new, count = s["ctx"].long(), s["new"].long(), s["count"].long()
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)]).clamp_max(tokens)
    new = starts[1:] - starts[:-1]
    old = ((ctx + page - 1) // page).clamp_max(width)
    need = ((ctx + new + page - 1) // page).clamp_max(width) - old
    base = need.cumsum(0) - need
    t = torch.arange(tokens, device=DEV)
    live = t < starts[-1]
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp_max(ctx.numel() - 1)
    pos = ctx[r] + t - starts[r]
    j = pos // page
    fresh, rank = j >= old[r], base[r] + j - old[r]
    taken = torch.where(rank < count, s["free"].long()[(count - 1 - rank).clamp(0, s["free"].numel() - 1)], -1)
    held = table.long()[r, j.clamp_max(width - 1)]
    at = torch.where(j >= width, -1, torch.where(fresh, taken, held))
    first = live & fresh & (pos % page == 0) & (j < width)
    table[r[first], j[first]] = at[first].to(torch.int32)
    slots = torch.where(live & (at >= 0), at * page + pos % page, -1)
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return {"starts": whole(starts), "requests": whole(torch.where(live, r, -1)), "positions": whole(torch.where(live, pos, 0)), "slots": whole(slots),
            "lens": whole(ctx + new), "count": whole((count - need.sum()).clamp_min(0)), "table": table}


def _plain_rope(s, c):
    q, k, v = (x.float() for x in _heads(s))
    r = c["rotary"]
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        y = x.clone()
        a, b = (slice(0, r, 2), slice(1, r, 2)) if c["layout"] == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y

    live = s["slots"] >= 0
    at = s["slots"][live].long()
    page, off = at // c["page"], at % c["page"]
    _plain_store(s["kc"], page, off, turned(k, s["kw"])[live], s["ks"])
    _plain_store(s["vc"], page, off, v[live], s["vs"])
    return {"q": turned(q, s["qw"]).to(DTYPES[c["dtype"]]), "k": s["kc"], "v": s["vc"]}


def _plain_store(cache, page, off, x, scale):
    if scale is None:
        cache[page, :, off] = x.to(cache.dtype)
    else:
        cache.view(torch.uint8)[page, :, off] = (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_rows(cache, page, off, scale):
    """Keys or values at those places in float32, [..., heads, dim]."""
    if scale is None:
        return cache[page, :, off].float()
    return cache.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).float() * scale[:, None]


def _plain_attend(s, c):
    n, h, g, d, page = c["requests"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    j = torch.arange(s["table"].shape[1] * page, device=DEV)
    at, off = s["table"][:, j // page].long().clamp_min(0), (j % page).expand(n, -1)
    lens = s["lens"][:, None]
    seen = (j < lens) & ((j >= lens - c["window"]) if c["window"] else (j >= 0))
    k = _plain_rows(s["kc"], at, off, s["ks"])  # [n, length, kv_heads, dim]
    x = torch.matmul(s["q"].float().view(n, g, h // g, d), k.permute(0, 2, 3, 1)) / math.sqrt(d)
    del k
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    v = _plain_rows(s["vc"], at, off, s["vs"]).masked_fill_(~seen[..., None, None], 0.0)
    y = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    out = {"out": y.view(n, h, d).to(DTYPES[c["dtype"]])}
    return {**out, "lse": (m + torch.log(total)).view(n, h)} if c["lse"] else out


def _plain_logprobs(s, c):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * (x - m), 0.0).sum(1, keepdim=True) / total
    out = {"logprobs": (x.gather(1, s["tokens"][:, None].long()) - m - log_total)[:, 0], "entropy": entropy[:, 0]}
    if c["top"]:
        top, ids = torch.sort(x, dim=1, descending=True, stable=True)
        out |= {"ids": ids[:, :c["top"]].to(torch.int32), "top": top[:, :c["top"]] - m - log_total}
    return out


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def exact(c, seed):
    if c["kind"] == "plan":
        return None  # whole numbers
    s = prepare(c, seed)
    if c["kind"] == "rope":
        return _exact_rope(s, c)
    if c["kind"] == "attend":
        return _exact_attend(s, c)
    x = s["logits"].double()
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    p = torch.exp(logp)
    out = {"logprobs": logp[torch.arange(c["rows"], device=DEV), s["tokens"].long()], "entropy": torch.special.entr(p).sum(1)}
    return {**out, "ids": None, "top": torch.topk(logp, c["top"], dim=1).values} if c["top"] else out


def _exact_rope(s, c):
    r, h, g, d = c["rotary"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().view(c["tokens"], h + 2 * g, d)
    for lo, hi, w in ((0, h, s["qw"]), (h, h + g, s["kw"])):
        if w is not None:
            x[:, lo:hi] *= w.double() / torch.sqrt(x[:, lo:hi].square().mean(2, keepdim=True) + 1e-6)
    if c["layout"] == "interleaved":
        z = torch.view_as_complex(x[:, :h + g, :r].reshape(c["tokens"], h + g, r // 2, 2).contiguous())
    else:
        z = torch.complex(x[:, :h + g, :r // 2].contiguous(), x[:, :h + g, r // 2:r].contiguous())
    z = z * torch.polar(torch.full_like(s["freq"], s["magnitude"]).expand(c["tokens"], -1), torch.outer(s["positions"].double(), s["freq"]))[:, None]
    x[:, :h + g, :r] = torch.view_as_real(z).flatten(2) if c["layout"] == "interleaved" else torch.cat([z.real, z.imag], 2)
    out = {"q": x[:, :h]}
    for name, lo, cache, scale in (("k", h, s["kc"], s["ks"]), ("v", h + g, s["vc"], s["vs"])):
        y = cache.double().transpose(1, 2).reshape(-1, g, d)
        live = (s["slots"] >= 0).nonzero()[:, 0]
        new = x[live, lo:lo + g]
        y[s["slots"][live].long()] = new if scale is None else (new / scale.double()[:, None]).clamp(-448, 448)
        out[name] = y.view(-1, c["page"], g, d).transpose(1, 2).contiguous()
    return out


def _exact_attend(s, c):
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros((c["requests"], h, d), dtype=torch.float64, device=DEV)
    lse = torch.full((c["requests"], h), -math.inf, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        if not n:
            continue
        lo = max(0, n - c["window"]) if c["window"] else 0
        pages = s["table"][i, lo // c["page"]:-(-n // c["page"])].long()
        skip = lo - lo // c["page"] * c["page"]
        k, v = (x[pages].double().transpose(0, 1).reshape(g, -1, d)[:, skip:skip + n - lo] for x in (s["kc"], s["vc"]))
        if s["ks"] is not None:
            k, v = k * s["ks"].double()[:, None, None], v * s["vs"].double()[:, None, None]
        x = torch.einsum("gud,gnd->gun", s["q"][i].double().view(g, h // g, d), k) * d ** -0.5
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        lse[i] = torch.logsumexp(x, 2).flatten()
        out[i] = torch.einsum("gun,gnd->gud", torch.softmax(x, 2), v).reshape(h, d)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(c):
    if c["kind"] == "plan":
        fresh = c["tokens"] / c["page"]
        return {"bytes": 16 * c["requests"] + 12 * c["tokens"] + 8 * fresh, "flops": c["tokens"]}
    if c["kind"] == "rope":
        t, h, g, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        return {"bytes": t * (2 * (2 * h + 2 * g) * d + 2 * g * d * BYTES[c["cache"]] + 8), "flops": t * (h + g) * (4 * d + 3 * c["rotary"])}
    if c["kind"] == "attend":
        seen = sum(min(n, c["window"]) if c["window"] else n for n in _lens(c))
        h, d = c["heads"], c["dim"]
        return {"bytes": seen * c["kv_heads"] * d * 2 * BYTES[c["cache"]] + c["requests"] * h * d * 4 + 4 * seen / c["page"], "flops": 4 * seen * h * d}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * BYTES[c["dtype"]] + c["rows"] * (12 + 8 * c["top"]), "flops": 5 * n}
