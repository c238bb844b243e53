"""More of the serving operators that the framework is timed on, and their plain forms.

What a serving step over a paged cache needs beside plan, write and attention:
heads rotated at positions of the program's own (``rotary``), the attention weight
that every cached key has received (``paged_key_weights``), the cache cut down to the
keys that received most (``paged_evict``), and the verification of drafted tokens
(``verify_drafts``). Sizes are those of the Qwen3-32B block (64 query heads on
8 key/value heads of 128, vocabulary 151936) and of the tests' smaller blocks, with contexts from
a hundred tokens to 128K.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
THETA, EPS = 1e6, 1e-6
FACTOR, ORIGINAL = 4.0, 32768  # a context of 32K positions stretched to 128K


def _rotary(name, tokens, heads, *, dim=128, part=None, interleaved=False, norm=False, scaling="none", dtype="bf16",
            furthest=32768):
    """Heads at positions up to ``furthest``; the first ``part`` values of a head are rotated."""
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "dim": dim, "part": part or dim,
            "interleaved": interleaved, "norm": norm, "scaling": scaling, "dtype": dtype, "furthest": furthest}


def _weights(name, requests, context, new, *, page=16, heads=64, kv_heads=8, dim=128, window=0):
    """Requests whose context and new lengths are spread over the two ranges."""
    return {"name": name, "kind": "weights", "requests": requests, "context_low": context[0], "context_high": context[1],
            "new_low": new[0], "new_high": new[1], "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window}


def _evict(name, requests, context, keep, recent, *, page=16, kv_heads=8, dim=128):
    """Requests of ``context`` tokens cut down to ``keep``, the last ``recent`` of them among it."""
    return {"name": name, "kind": "evict", "requests": requests, "context_low": context[0], "context_high": context[1],
            "new_low": 0, "new_high": 0, "page": page, "kv_heads": kv_heads, "dim": dim, "keep": keep, "recent": recent}


def _verify(name, requests, drafts, vocab, *, model=True, dtype="f32"):
    """Requests with ``drafts`` drafted tokens each, drawn by a smaller model, or (``model`` False) looked up."""
    return {"name": name, "kind": "verify", "requests": requests, "drafts_low": drafts[0], "drafts_high": drafts[1],
            "vocab": vocab, "model": model, "dtype": dtype}


def listed():
    return [
        # Query and key heads of a decode step of 16 requests, far into long contexts: the smallest call.
        _rotary("rotary_decode_16", 16, 72, norm=True, scaling="yarn", furthest=131072),
        # Those of a prefill of 8 prompts of 1024 tokens.
        _rotary("rotary_prefill_8x1024", 8192, 72, furthest=1024),
        # A ragged chunk in FP32, pairs of neighbours, half of each head rotated.
        _rotary("rotary_part_interleaved", 3001, 40, part=64, interleaved=True, scaling="linear", dtype="f32"),
        # One decode step of 64 requests of ragged context, the ordinary serving load.
        _weights("weights_decode_64", 64, (100, 8100), (1, 1)),
        # A decode step over four contexts of 128K tokens.
        _weights("weights_decode_long_4", 4, (131000, 131000), (1, 1), page=64),
        # A 2048-token chunk of a long prompt, 16K tokens of which are cached.
        _weights("weights_chunk_2048", 1, (16384, 16384), (2048, 2048)),
        # A few requests a page's tokens over their budget, as a decoding server finds them.
        _evict("evict_steady_8", 8, (1040, 1040), 1024, 64),
        # A server's requests cut to 2048 tokens; the shorter ones stay whole.
        _evict("evict_ragged_64", 64, (100, 8100), 2048, 256),
        # Four prompts of 128K tokens cut to a quarter after their prefill.
        _evict("evict_prompts_4", 4, (131000, 131000), 32768, 512, page=64),
        # One request with four drafted tokens.
        _verify("verify_1", 1, (4, 4), 151936),
        # A decode batch, some requests without drafts.
        _verify("verify_ragged_64", 64, (0, 7), 151936),
        # Drafts looked up in the prompt (no distribution of their own), bf16 probabilities.
        _verify("verify_lookup_200", 200, (1, 3), 32001, model=False, dtype="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rotary", "weights", "weights", "evict", "evict", "verify"))
    if kind == "rotary":
        dim = rng.choice((64, 80, 96, 128, 128, 256))
        norm = dim in (64, 128, 256) and rng.random() < 0.3
        heads = rng.choice((8, 10, 24, 40, 72))
        return _rotary("", _log(rng, 1, 8192 * 72 * 128 // (heads * dim) // 2), heads, dim=dim,
                       part=rng.choice((dim, dim, 32, dim // 2)), interleaved=rng.random() < 0.4, norm=norm,
                       scaling=rng.choice(("none", "linear", "ntk", "yarn")), dtype=rng.choice(("bf16", "bf16", "f32")),
                       furthest=_log(rng, 100, 1 << 20))
    if kind == "verify":
        vocab, most = _log(rng, 1000, 151936), 64 * 151936
        requests = _log(rng, 1, min(512, most // vocab))
        low = rng.randint(0, 4)
        return _verify("", requests, (low, low + rng.randint(0, 4)), vocab, model=rng.random() < 0.7,
                       dtype=rng.choice(("f32", "f32", "bf16")))
    page, dim = rng.choice((8, 16, 32, 64, 128)), rng.choice((64, 128, 128))
    if kind == "evict":
        kv_heads, requests = rng.choice((2, 4, 8)), _log(rng, 1, 128)
        high = _log(rng, 32, min(131000, 400000 // requests))
        keep = _log(rng, 8, high)
        return _evict("", requests, (rng.randint(1, high), high), keep, rng.choice((0, rng.randint(0, keep // 4), keep)) if
                      keep < 2000 else rng.randint(0, 600), page=page, kv_heads=kv_heads, dim=dim)
    heads, kv_heads = rng.choice(((64, 8), (16, 8), (8, 2), (8, 8), (40, 8)))
    shape = dict(page=page, heads=heads, kv_heads=kv_heads, dim=dim)
    if rng.random() < 0.5:  # decode
        requests = _log(rng, 1, 128)
        high = _log(rng, 16, min(131000, 400000 // requests))
        return _weights("", requests, (rng.randint(0, high), high), (1, rng.choice((1, 1, 2, 5))),
                        window=rng.choice((0, 0, _log(rng, 16, 4096))), **shape)
    requests = _log(rng, 1, 16)
    new = _log(rng, 16, 1600 // requests)
    return _weights("", requests, (0, _log(rng, 16, 16000 // requests)), (1, new),
                    window=rng.choice((0, 0, _log(rng, 16, 2048))), **shape)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _spread(count, low, high, phase):
    """``count`` lengths in low .. high, spread evenly, in a mixed order."""
    at = (torch.arange(count, dtype=torch.float64) * 0.6180339887498949 + phase) % 1.0
    return (low + (at * (high - low + 1)).long()).clamp(max=high)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _rotary_inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    heads, dim, part = case["heads"], case["dim"], case["part"]
    # the front columns of one projection's output: query and key heads, value heads behind them
    heads_and_values = _randn(g, case["tokens"], heads + 8, dim).to(_dtype(case))
    half = part // 2
    f = THETA ** (-torch.arange(half, dtype=torch.float64) * 2 / part)
    amplitude = 1.0
    if case["scaling"] == "linear":  # every position moves closer
        f = f / FACTOR
    elif case["scaling"] == "ntk":  # a larger base: the slowest pair alone is stretched by the whole factor
        f = (THETA * FACTOR ** (part / (part - 2))) ** (-torch.arange(half, dtype=torch.float64) * 2 / part)
    elif case["scaling"] == "yarn":  # pairs that turn often stay, slow ones are stretched, a ramp between
        def pair(turns):
            return part * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))

        low, high = max(0, math.floor(pair(32))), min(part - 1, math.ceil(pair(1)))
        ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / FACTOR * ramp
        amplitude = 0.1 * math.log(FACTOR) + 1
    positions = torch.randint(0, case["furthest"], (case["tokens"],), device=DEVICE, generator=g, dtype=torch.int32)
    return {"case": case, "x": heads_and_values[:, :heads], "positions": positions, "frequencies": f.to(DEVICE),
            "amplitude": amplitude,
            "norm": (1 + 0.1 * _randn(g, dim)).to(torch.bfloat16) if case["norm"] else None}


def _tables(g, case, length):
    """Block tables of shuffled pages, -1 behind each request's last page."""
    pages = -(-length // case["page"])
    total = int(pages.sum())
    order = torch.randperm(total + 5, device=DEVICE, generator=g).to(torch.int32)
    at = torch.arange(max(1, int(pages.max())), device=DEVICE)[None, :]
    held = pages.to(DEVICE)
    first = (held.cumsum(0) - held)[:, None]
    return torch.where(at < held[:, None], order[(first + at).clamp(max=total + 4)], -1).to(torch.int32), total + 5


def _lengths(case):
    """Context and new lengths of every request (on the host)."""
    return (_spread(case["requests"], case["context_low"], case["context_high"], 0.37),
            _spread(case["requests"], case["new_low"], case["new_high"], 0.81))


def _cache_inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    context, new = _lengths(case)
    tables, num_pages = _tables(g, case, context + new)
    s = {"case": case, "context": context.to(DEVICE, torch.int32), "new": new.to(DEVICE, torch.int32), "tables": tables,
         "num_pages": num_pages, "used": int(new.sum()), "most_new": max(1, int(new.max())),
         "longest": int((context + new).max()), "tokens": max(16, -(-int(new.sum()) // 16) * 16)}
    cache = (num_pages, case["page"], case["kv_heads"], case["dim"])
    s["k_cache"] = _randn(g, *cache).to(torch.bfloat16)
    # what keys have received so far: a few of them most of it
    received = (_randn(g, num_pages, case["kv_heads"], case["page"]) * 1.5 - 3).exp_()
    if case["kind"] == "weights":
        s["weights"] = received
        # normalised heads: scores of a standard deviation of about 1.5
        s["q"] = (1.5 * _randn(g, s["tokens"], case["heads"], case["dim"])).to(torch.bfloat16)
        s["lse"] = _row_sums(s)
        return s
    s["v_cache"] = _randn(g, *cache).to(torch.bfloat16)
    s["received"], s["weights"] = received, torch.empty_like(received)
    return s


def _verify_inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    vocab, requests = case["vocab"], case["requests"]
    new = _spread(requests, case["drafts_low"], case["drafts_high"], 0.81) + 1
    rows = int(new.sum())
    logits = 3 * _randn(g, rows, vocab)
    target = torch.softmax(logits, dim=-1).to(_dtype(case))
    # a smaller model's logits are the large one's but for some noise
    guess = torch.softmax(logits + 0.7 * _randn(g, rows, vocab), dim=-1).to(_dtype(case))
    del logits
    s = {"case": case, "target": target, "draft": guess if case["model"] else None, "new": new.to(DEVICE, torch.int32),
         "rows": rows, "most_new": int(new.max())}
    # row i + 1 holds the token that was drawn from row i's guess
    noise = torch.rand(rows, vocab, device=DEVICE, generator=g).clamp_(min=1e-9)
    s["step_tokens"] = torch.roll((guess.float() / -noise.log()).argmax(-1), 1).to(torch.int32)
    s["accept"] = torch.rand(rows, device=DEVICE, generator=g)
    s["sample"] = torch.rand(requests, device=DEVICE, generator=g)
    return s


def _plan(s):
    import strassen_tpu_amd as smx

    if s["case"]["kind"] == "verify":  # a step's plan; its cache is not read here
        lens = torch.zeros_like(s["new"])
        table = torch.arange(lens.numel(), device=DEVICE, dtype=torch.int32)[:, None].contiguous()
        return smx.paged_plan(lens, s["new"], table, page_size=16, num_pages=lens.numel(), tokens=s["rows"],
                              max_new=s["most_new"])
    return smx.paged_plan(s["context"], s["new"], s["tables"], page_size=s["case"]["page"], num_pages=s["num_pages"],
                          tokens=s["tokens"], max_new=s["most_new"])


def prepare(case, seed):
    kind = case["kind"]
    if kind == "rotary":
        return _rotary_inputs(case, seed)
    s = _verify_inputs(case, seed) if kind == "verify" else _cache_inputs(case, seed)
    if own and kind != "evict":  # one plan serves every layer of a step
        s["plan"] = _plan(s)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _own_pass(s):
    import strassen_tpu_amd as smx

    case, kind = s["case"], s["case"]["kind"]
    if kind == "rotary":
        return smx.rotary(s["x"], s["positions"], s["frequencies"], interleaved=case["interleaved"],
                          amplitude=s["amplitude"], norm=s["norm"], eps=EPS)
    if kind == "weights":
        smx.paged_key_weights(s["q"], s["k_cache"], s["weights"], s["plan"], s["lse"], window=case["window"] or None)
        return s["weights"]
    if kind == "evict":
        s["weights"].copy_(s["received"])  # what was received since the pass before
        lens = smx.paged_evict(s["k_cache"], s["v_cache"], s["weights"], s["context"], s["tables"], case["keep"],
                               recent=case["recent"])
        return [lens, s["k_cache"], s["v_cache"], s["weights"]]
    return list(smx.verify_drafts(s["target"], s["step_tokens"], s["plan"], s["accept"], s["sample"], draft=s["draft"]))


def _plain_rotary(s):
    case, x = s["case"], s["x"].float()
    part = case["part"]
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
    angle = s["positions"].double()[:, None] * s["frequencies"]  # far positions: in 64 bits
    cos, sin = (s["amplitude"] * f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    turned, rest = x[..., :part], x[..., part:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned.chunk(2, dim=-1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1).to(s["x"].dtype)


def _rows_of(new, tokens):
    """The request of each row, the row's place among its request's and the rows' starts."""
    new = new.long()
    ends = new.cumsum(0)
    rows = torch.arange(tokens, device=DEVICE)
    request = torch.searchsorted(ends, rows, right=True).clamp(max=new.numel() - 1)
    return request, rows - (ends - new)[request], ends - new


def _scores(s):
    """Masked scores [requests, kv_heads, most_new, group, length] of all requests at once, padded to the longest."""
    case, q, used = s["case"], s["q"], s["used"]
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    requests, most, context = case["requests"], s["most_new"], s["context"].long()
    request, place, _ = _rows_of(s["new"], used)
    rows = torch.zeros(requests, most, heads, dim, device=DEVICE)
    rows[request, place] = q[:used].float()
    rows = rows.view(requests, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(
        requests * kv_heads, -1, dim)
    length = s["tables"].shape[1] * page
    keys = s["k_cache"][s["tables"].long().clamp(min=0)].view(requests, length, kv_heads, dim).permute(0, 2, 3, 1).float()
    scores = torch.bmm(rows, keys.reshape(requests * kv_heads, dim, length)).mul_(dim ** -0.5)
    del keys
    key = torch.arange(length, device=DEVICE)
    own_key = context[:, None] + torch.arange(most, device=DEVICE)[None, :]
    seen = key <= own_key[..., None]
    if case["window"]:
        seen &= key > own_key[..., None] - case["window"]
    seen &= (torch.arange(most, device=DEVICE)[None, :] < s["new"][:, None])[..., None]
    scores = scores.view(requests, kv_heads, most, heads // kv_heads, length)
    return scores.masked_fill_(~seen[:, None, :, None, :], float("-inf")), request, place


def _row_sums(s):
    """What the step's attention hands on: the logarithm of each row's sum of exponentials, [tokens, heads]."""
    scores, request, place = _scores(s)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    sums = scores.sub_(top).exp_().sum(-1, keepdim=True).log().add_(top)[..., 0]
    lse = torch.zeros(s["tokens"], s["case"]["heads"], device=DEVICE)
    lse[:s["used"]] = sums.permute(0, 2, 1, 3).flatten(2)[request, place]
    return lse


def _plain_weights(s):
    case, used = s["case"], s["used"]
    requests, kv_heads, page, most = case["requests"], case["kv_heads"], case["page"], s["most_new"]
    scores, request, place = _scores(s)
    lse = torch.zeros(requests, most, case["heads"], device=DEVICE)
    lse[request, place] = s["lse"][:used]
    lse = lse.view(requests, most, kv_heads, -1).permute(0, 2, 1, 3)[..., None]
    found = scores.sub_(lse).exp_().sum((2, 3))  # [requests, kv_heads, length]
    context, new = s["context"].long()[:, None], s["new"].long()[:, None]
    key = torch.arange(found.shape[-1], device=DEVICE)[None, :]
    # keys behind a request's last, and requests that sit the step out, repeat the request's first key
    at = torch.where((key < context + new) & (new > 0), key, 0)
    slot_page, slot = s["tables"].long().gather(1, at // page).clamp(min=0), at % page
    before = s["weights"][slot_page, :, slot]  # [requests, length, kv_heads]
    before = before.masked_fill(((at >= context) & (new > 0))[..., None], 0)
    s["weights"][slot_page, :, slot] = before + found.transpose(1, 2).gather(1, at[..., None].expand(-1, -1, kv_heads))
    return s["weights"]


def _plain_evict(s):
    case, page, recent = s["case"], s["case"]["page"], min(s["case"]["recent"], s["case"]["keep"])
    need = case["keep"] - recent
    s["weights"].copy_(s["received"])
    n = s["context"].long()[:, None]  # [requests, 1]
    index = torch.arange(s["longest"], device=DEVICE)[None, :]
    known = torch.where(index < n, index, 0)
    slot_page, slot = s["tables"].long().gather(1, known // page), known % page
    received = s["weights"][slot_page, :, slot].transpose(1, 2)  # [requests, kv_heads, length]
    old, index = (index < n - recent)[:, None], index[:, None]
    order = received.masked_fill(~old, float("-inf")).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, torch.arange(s["longest"], device=DEVICE).expand_as(order))
    cut = (n > case["keep"])[..., None]
    stays = old & (rank < need)
    hole, mover = cut & (index < need) & ~stays, cut & (index >= need) & stays
    # the j-th hole takes the j-th survivor that lies behind
    movers = torch.zeros_like(order).scatter_(-1, torch.where(mover, mover.cumsum(-1) - 1, s["longest"] - 1),
                                              torch.where(mover, index, 0))
    source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), index.expand_as(order))
    source = torch.where(cut & (index >= need) & (index < case["keep"]), index + (n[..., None] - case["keep"]), source)
    source = torch.where(cut & (index < case["keep"]), source, index)[..., :case["keep"]]
    width = source.shape[-1]
    inside = index[..., :width] < n[..., None]  # others repeat the request's first token
    source = torch.where(inside, source, source[..., :1])
    target = torch.where(inside, index[..., :width], 0).expand_as(source)
    heads = torch.arange(case["kv_heads"], device=DEVICE)[None, :, None]
    pages = s["tables"].long()[:, None].expand(-1, case["kv_heads"], -1)
    from_page, to_page = pages.gather(-1, source // page), pages.gather(-1, target // page)
    for cache in (s["k_cache"], s["v_cache"]):
        cache[to_page, target % page, heads] = cache[from_page, source % page, heads]
    s["weights"][to_page, heads, target % page] = s["weights"][from_page, heads, source % page]
    return [s["context"].clamp(max=case["keep"]), s["k_cache"], s["v_cache"], s["weights"]]


def _plain_verify(s):
    target, draft, tokens, new = s["target"], s["draft"], s["step_tokens"].long(), s["new"].long()
    request, place, starts = _rows_of(s["new"], s["rows"])
    drafted = torch.roll(tokens, -1)  # the token behind each row
    p = target.gather(1, drafted[:, None])[:, 0].double()
    q = draft.gather(1, drafted[:, None])[:, 0].double() if draft is not None else torch.ones_like(p)
    checked = place + 1 < new[request]
    refused = checked & ~(s["accept"].double() * q < p)
    accepted = (new - 1).scatter_reduce(0, request, torch.where(refused, place, s["most_new"]), "amin")
    row, whole = starts + accepted, accepted + 1 == new
    p = target[row].double()
    if draft is not None:
        rest = (p - draft[row].double().masked_fill(whole[:, None], 0)).clamp(min=0)
    else:
        mine = torch.arange(p.shape[1], device=DEVICE) == drafted[row][:, None]
        rest = p.masked_fill(mine & ~whole[:, None], 0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    sums = rest.cumsum(-1)
    fits = (sums > s["sample"].double()[:, None] * rest.sum(-1, keepdim=True)) & (rest > 0)
    index = torch.arange(p.shape[1], device=DEVICE)
    last = torch.where(rest > 0, index, -1).amax(-1)
    drawn = torch.where(fits.any(-1), torch.where(fits, index, p.shape[1]).amin(-1), last)
    out = torch.where(place < accepted[request], drafted, torch.where(place == accepted[request], drawn[request], -1))
    return [out.to(torch.int32), (accepted + 1).to(torch.int32)]


def run(state):
    if own:
        return _own_pass(state)
    return {"rotary": _plain_rotary, "weights": _plain_weights, "evict": _plain_evict,
            "verify": _plain_verify}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        size = 2 if case["dtype"] == "bf16" else 4
        turned = case["tokens"] * case["heads"] * case["part"]
        return {"bytes": 2 * size * values + 4 * case["tokens"], "flops": 3 * turned + (4 * values if case["norm"] else 0)}
    if kind == "verify":
        size = 2 if case["dtype"] == "bf16" else 4
        rows = case["requests"] * (2 if case["model"] and case["drafts_high"] else 1)
        return {"bytes": rows * case["vocab"] * size + 12 * case["requests"] * (1 + case["drafts_high"]),
                "flops": 3 * case["requests"] * case["vocab"]}
    context, new = (x.double() for x in _lengths(case))
    kv = case["kv_heads"] * case["dim"]
    if kind == "evict":
        recent = min(case["recent"], case["keep"])
        need = case["keep"] - recent
        n = context[context > case["keep"]]
        # survivors fall anywhere among the older tokens, which are a share of them behind the places kept
        moved = need * (1 - need / (n - recent)) + torch.minimum(torch.full_like(n, recent), n)
        return {"bytes": float(4 * case["kv_heads"] * n.sum() + (8 * kv + 8 * case["kv_heads"]) * moved.sum()) + 8 * case["requests"],
                "flops": float(case["kv_heads"] * n.sum()) + case["requests"]}
    tokens, length = float(new.sum()), context + new
    pairs = new * context + new * (new + 1) / 2
    if case["window"]:
        w = torch.tensor(float(case["window"]), dtype=torch.float64)
        low, ramp = torch.minimum(context, w), torch.minimum(length, w) - torch.minimum(context, w)
        pairs = ramp * low + ramp * (ramp + 1) / 2 + (new - ramp) * w
        length = torch.minimum(length, new + w - 1)
    heads = case["heads"]
    return {"bytes": float(tokens * heads * (2 * case["dim"] + 4)
                           + (2 * kv + 8 * case["kv_heads"] + 4 / case["page"]) * length.sum()),
            "flops": float(2 * heads * case["dim"] * pairs.sum())}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None  # whole numbers
    if kind == "rotary":
        s = _rotary_inputs(case, seed)
        part, half = case["part"], case["part"] // 2
        out = s["x"].double().clone()
        if s["norm"] is not None:
            out = out / torch.sqrt((out * out).sum(-1, keepdim=True) / case["dim"] + EPS) * s["norm"].double()
        turned = torch.view_as_complex(
            (out[..., :part].reshape(*out.shape[:2], half, 2) if case["interleaved"]
             else torch.stack((out[..., :half], out[..., half:part]), -1)).contiguous())
        turned = turned * torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device=DEVICE).expand(
            case["tokens"], half).contiguous(), s["positions"].double()[:, None] * s["frequencies"])[:, None]
        both = torch.view_as_real(turned)
        out[..., :part] = both.flatten(-2) if case["interleaved"] else torch.cat((both[..., 0], both[..., 1]), -1)
        return out
    s = _cache_inputs(case, seed)
    context, new = _lengths(case)
    page = case["page"]
    if kind == "evict":
        k_cache, v_cache, weights = s["k_cache"].double(), s["v_cache"].double(), s["received"].double()
        lens, keep, recent = s["context"].clone(), case["keep"], min(case["recent"], case["keep"])
        for b, n in enumerate(context.tolist()):
            if n <= keep:
                continue
            lens[b] = keep
            at = torch.arange(n, device=DEVICE)
            pages, slots = s["tables"][b].long()[at // page], at % page
            for h in range(case["kv_heads"]):
                mine = weights[pages, h, slots]
                # by weight, then by index
                best = torch.sort(-mine[:n - recent], stable=True).indices[:keep - recent].sort().values
                stay, come = best[best < keep - recent], best[best >= keep - recent]
                free = torch.ones(keep - recent, dtype=torch.bool, device=DEVICE)
                free[stay] = False
                to = torch.cat((free.nonzero()[:, 0], at[keep - recent:keep]))
                of = torch.cat((come, at[n - recent:]))
                for cache in (k_cache, v_cache):
                    cache[pages[to], slots[to], h] = cache[pages[of], slots[of], h]
                weights[pages[to], h, slots[to]] = mine[of]
        return [lens, k_cache, v_cache, weights]
    weights, row, ratio = s["weights"].double(), 0, case["heads"] // case["kv_heads"]
    for b, (c, w) in enumerate(zip(context.tolist(), new.tolist())):
        if not w:
            continue
        at = torch.arange(c + w, device=DEVICE)
        pages, slots = s["tables"][b].long()[at // page], at % page
        mine = at[c:, None]
        hidden = at[None, :] > mine
        if case["window"]:
            hidden = hidden | (at[None, :] <= mine - case["window"])
        weights[pages[c:], :, slots[c:]] = 0
        for h in range(case["kv_heads"]):
            keys, found = s["k_cache"][pages, slots, h].double(), torch.zeros(c + w, dtype=torch.float64, device=DEVICE)
            for j in range(h * ratio, (h + 1) * ratio):
                score = s["q"][row:row + w, j].double() @ keys.t() / math.sqrt(case["dim"])
                score = torch.exp(score - s["lse"][row:row + w, j].double()[:, None])
                found += score.masked_fill(hidden, 0).sum(0)
            weights[pages, h, slots] += found
        row += w
    return weights
