"""The serving operators that the framework is timed on, and their plain forms.

A serving step of a decoder block: requests of ragged lengths append new
tokens to a paged key/value cache (``paged_plan`` lays out pages and rows,
``paged_write`` normalises, rotates and stores the heads), attend over it
(``paged_attention``) and go through projections whose weights are kept in 4
bits (``int4_matmul``). Sizes are those of the Qwen3-32B block (64 query heads on
8 key/value heads of 128, hidden 5120, ffn 25600) and of the tests' smaller
blocks, with contexts from a hundred tokens to 128K.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
THETA, EPS = 1e6, 1e-6


def _serve(kind, name, requests, context, new, *, page=16, heads=64, kv_heads=8, dim=128, window=0, short=0.0):
    """Requests whose context and new lengths are spread over the two ranges.
    ``short``: the share of the pages that the step needs and the free list lacks."""
    return {"name": name, "kind": kind, "requests": requests, "context_low": context[0], "context_high": context[1],
            "new_low": new[0], "new_high": new[1], "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "short": short}


def _product(name, m, k, n, *, group=128, epilogue="none", zeros=True):
    return {"name": name, "kind": "int4", "m": m, "k": k, "n": n, "group": group, "epilogue": epilogue, "zeros": zeros}


def listed():
    return [
        # One decode step of 16 requests: the smallest plan, all latency.
        _serve("plan", "plan_decode_16", 16, (100, 4000), (1, 1)),
        # A large server's step: 2048 requests, most of them decoding, some idle
        # or appending a piece of a prompt, and too few free pages for all.
        _serve("plan", "plan_ragged_2048", 2048, (0, 8000), (0, 63), short=0.1),
        # The heads of one decode step of 16 requests.
        _serve("write", "write_decode_16", 16, (100, 4000), (1, 1)),
        # The heads of a prefill of 8 prompts of 1024 tokens.
        _serve("write", "write_prefill_8x1024", 8, (0, 0), (1024, 1024), page=64),
        # One request's decode step early in its answer, the smallest attention call.
        _serve("attention", "attention_decode_1", 1, (1000, 1000), (1, 1)),
        # A decode step of 64 requests of ragged context, the ordinary serving load.
        _serve("attention", "attention_decode_64", 64, (100, 8100), (1, 1)),
        # A decode step over four contexts of 128K tokens.
        _serve("attention", "attention_decode_long_4", 4, (131000, 131000), (1, 1), page=64),
        # A 2048-token chunk of a long prompt, 16K tokens of which are cached.
        _serve("attention", "attention_chunk_2048", 1, (16384, 16384), (2048, 2048)),
        # Pieces of prompts of ragged length beside decoding requests, sliding window.
        _serve("attention", "attention_ragged_window", 12, (0, 5000), (1, 700), page=32, window=1024),
        # The down projection of one decoding request, its K the longest of the model's.
        _product("int4_down_1", 1, 25600, 5120, epilogue="residual_add"),
        # The gate|up projection of a decode step of 16 requests.
        _product("int4_gate_up_16", 16, 5120, 51200, epilogue="swiglu"),
        # The query projection of a larger decode batch of ragged size, small groups.
        _product("int4_query_61", 61, 5120, 8192, group=32, zeros=False),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("plan", "write", "attention", "attention", "attention", "int4", "int4"))
    if kind == "int4":
        group = rng.choice((32, 64, 128))
        n = _log(rng, 200, 51200)
        epilogue = rng.choice(("none", "bias_add", "residual_add", "swiglu"))
        return _product("", _log(rng, 1, 64), group * _log(rng, 4, 25600 // group),
                        n + n % 2 if epilogue == "swiglu" else n, group=group, epilogue=epilogue,
                        zeros=rng.random() < 0.5)
    page = rng.choice((8, 16, 32, 64, 128))
    heads, kv_heads = rng.choice(((64, 8), (16, 8), (8, 2), (8, 8), (40, 8)))
    dim = rng.choice((64, 128, 128))
    shape = dict(page=page, heads=heads, kv_heads=kv_heads, dim=dim)
    if kind == "plan":
        requests = _log(rng, 1, 2048)
        return _serve(kind, "", requests, (0, _log(rng, 16, 8000)), (rng.randint(0, 1), _log(rng, 1, 63)),
                      short=rng.choice((0.0, 0.0, 0.2)), **shape)
    if kind == "write":
        requests, most = _log(rng, 1, 64), 8192
        return _serve(kind, "", requests, (0, _log(rng, 16, 4000)), (1, _log(rng, 1, most // requests)), **shape)
    if rng.random() < 0.5:  # decode
        requests = _log(rng, 1, 128)
        high = _log(rng, 16, min(131000, 400000 // requests))
        return _serve(kind, "", requests, (rng.randint(0, high), high), (1, rng.choice((1, 1, 2, 5))), **shape)
    requests = _log(rng, 1, 16)
    new = _log(rng, 16, 1600 // requests)
    return _serve(kind, "", requests, (0, _log(rng, 16, 16000 // requests)), (1, new),
                  window=rng.choice((0, 0, _log(rng, 16, 2048))), **shape)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _spread(count, low, high, phase):
    """``count`` lengths in low .. high, spread evenly, in a mixed order."""
    at = (torch.arange(count, dtype=torch.float64) * 0.6180339887498949 + phase) % 1.0
    return (low + (at * (high - low + 1)).long()).clamp(max=high)


def _lengths(case):
    """Context and new lengths of every request (on the host)."""
    return (_spread(case["requests"], case["context_low"], case["context_high"], 0.37),
            _spread(case["requests"], case["new_low"], case["new_high"], 0.81))


def _tables(g, case, context, new):
    """Block tables of shuffled pages, -1 behind each request's last page; for a
    plan only the contexts' pages, and the others as the free list."""
    page = case["page"]
    pages = -(-(context if case["kind"] == "plan" else context + new) // page)
    total = int(((context + new + page - 1) // page).sum())
    num_pages = total + 5
    order = torch.randperm(num_pages, device=DEVICE, generator=g).to(torch.int32)
    width = max(1, int((-(-(context + new) // page)).max()))
    at = torch.arange(width, device=DEVICE)[None, :]
    held = pages.to(DEVICE)
    first = (held.cumsum(0) - held)[:, None]
    tables = torch.where(at < held[:, None], order[(first + at).clamp(max=num_pages - 1)], -1).to(torch.int32)
    lack = int(case["short"] * (total - int(pages.sum())))
    return tables, num_pages, order[int(pages.sum()):total - lack].contiguous()


def _randn(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32)


def _serve_inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    context, new = _lengths(case)
    tables, num_pages, free = _tables(g, case, context, new)
    s = {"case": case, "context": context.to(DEVICE, torch.int32), "new": new.to(DEVICE, torch.int32),
         "tables": tables, "num_pages": num_pages, "free": free, "used": int(new.sum()), "most_new": max(1, int(new.max())),
         # rows come in whole groups of 16, as the projections take them
         "tokens": max(16, -(-int(new.sum()) // 16) * 16)}
    if case["kind"] == "plan":
        return s
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    cache = (num_pages, case["page"], kv_heads, dim)
    s["k_cache"], s["v_cache"] = _randn(g, *cache).to(torch.bfloat16), _randn(g, *cache).to(torch.bfloat16)
    if case["kind"] == "attention":
        # normalised heads: scores of a standard deviation of about 1.5
        s["q"] = (1.5 * _randn(g, s["tokens"], heads, dim)).to(torch.bfloat16)
        return s
    # one projection's output, its columns the query, key and value heads
    qkv = _randn(g, s["tokens"], heads + 2 * kv_heads, dim).to(torch.bfloat16)
    s["q"], s["k"], s["v"] = qkv.split((heads, kv_heads, kv_heads), dim=1)
    s["q_scale"], s["k_scale"] = ((1 + 0.1 * _randn(g, dim)).to(torch.bfloat16) for _ in range(2))
    angle = torch.arange(tables.shape[1] * case["page"], device=DEVICE, dtype=torch.float64)[:, None] / THETA ** (
        torch.arange(0, dim, 2, device=DEVICE, dtype=torch.float64) / dim)
    s["cos"], s["sin"] = torch.cos(angle).to(torch.bfloat16), torch.sin(angle).to(torch.bfloat16)
    return s


def _product_inputs(case, seed):
    """Codes of normal weights over their group's range, scales of a projection ~ N(0, 0.02)."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
    codes = (_randn(g, k, n) * 2.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    scales = (0.0075 * (1 + 0.2 * _randn(g, groups, n))).to(torch.bfloat16)
    zeros = (_randn(g, groups, n) * 0.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8) if case["zeros"] else None
    s = {"case": case, "x": _randn(g, m, k).to(torch.bfloat16), "codes": codes, "scales": scales, "zeros": zeros,
         "extra": None}
    if case["epilogue"] == "residual_add":
        s["extra"] = _randn(g, m, n).to(torch.bfloat16)
    if case["epilogue"] == "bias_add":
        s["extra"] = _randn(g, n).to(torch.bfloat16)
    return s


def _plan(s):
    import strassen_tpu_amd as smx

    case = s["case"]
    return smx.paged_plan(s["context"], s["new"], s["tables"], page_size=case["page"], num_pages=s["num_pages"],
                          tokens=s["tokens"], max_new=s["most_new"],
                          free_pages=s["free"] if case["kind"] == "plan" else None)


def prepare(case, seed):
    if case["kind"] == "int4":
        s = _product_inputs(case, seed)
        if own:  # a program keeps its weights laid out, not as codes
            import strassen_tpu_amd as smx

            s["w"] = smx.int4_weight_layout(s.pop("codes"), s.pop("scales"), s.pop("zeros"), group=case["group"],
                                            epilogue="swiglu" if case["epilogue"] == "swiglu" else None)
        return s
    s = _serve_inputs(case, seed)
    if own and case["kind"] != "plan":  # one plan serves every layer of a step
        s["plan"] = _plan(s)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _own_pass(s):
    import strassen_tpu_amd as smx

    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        plan = _plan(s)
        return [plan.starts, plan.positions, plan.slots, plan.status, plan.pages_needed, s["tables"]]
    if kind == "write":
        q = smx.paged_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["plan"], q=s["q"], rope_cos=s["cos"],
                            rope_sin=s["sin"], q_scale=s["q_scale"], k_scale=s["k_scale"], eps=EPS)
        return [q, s["k_cache"], s["v_cache"]]
    if kind == "attention":
        return smx.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["plan"], window=case["window"] or None)
    epilogue = case["epilogue"]
    extra = {"residual_add": {"residual": s["extra"]}, "bias_add": {"bias": s["extra"]}}.get(epilogue, {})
    return smx.int4_matmul(s["x"], s["w"], epilogue=None if epilogue == "none" else epilogue, **extra)


def _rows_of(s):
    """The request of each row and the row's place among its request's."""
    new = s["new"].long()
    ends = new.cumsum(0)
    rows = torch.arange(s["tokens"], device=DEVICE)
    request = torch.searchsorted(ends, rows, right=True)
    inside = request < new.numel()
    request = request.clamp(max=new.numel() - 1)
    return request, rows - (ends - new)[request], inside, ends


def _plain_plan(s):
    page, tables, free = s["case"]["page"], s["tables"], s["free"]
    context, new = s["context"].long(), s["new"].long()
    request, place, inside, ends = _rows_of(s)
    first_new = (context + page - 1) // page  # pages that the context holds
    need = torch.where(new > 0, (context + new + page - 1) // page - first_new, 0)
    upto = need.cumsum(0)
    admitted = (need == 0) | (upto <= free.numel())
    status = torch.where(admitted, 0, 3).to(torch.int32)
    used = torch.where(admitted, upto, 0).max().reshape(1).to(torch.int32)
    # the new pages of the admitted requests, by columns of the table
    at = torch.arange(tables.shape[1], device=DEVICE)[None, :] - first_new[:, None]
    taken = (at >= 0) & (at < need[:, None]) & admitted[:, None]
    source = ((upto - need)[:, None] + at).clamp(0, max(0, free.numel() - 1))
    if free.numel():
        tables.copy_(torch.where(taken, free[source], tables))
    covered = inside & admitted[request]
    position = torch.where(covered, context[request] + place, -1)
    known = position.clamp(min=0)
    slot = tables[request, (known // page).clamp(max=tables.shape[1] - 1)].long() * page + known % page
    starts = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEVICE), ends)).to(torch.int32)
    return [starts, position.to(torch.int32), torch.where(covered, slot, -1), status, used, tables]


def _norm_rotate(x, scale, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * scale.float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(torch.bfloat16)


def _plain_write(s):
    page, used = s["case"]["page"], s["used"]
    request, place, _, _ = _rows_of(s)
    position = (s["context"].long()[request] + place)[:used]
    slot = s["tables"][request[:used], position // page].long() * page + position % page
    cos, sin = s["cos"].float()[position][:, None, :], s["sin"].float()[position][:, None, :]
    q = torch.zeros(s["q"].shape, dtype=torch.bfloat16, device=DEVICE)
    q[:used] = _norm_rotate(s["q"][:used], s["q_scale"], cos, sin)
    s["k_cache"].flatten(0, 1)[slot] = _norm_rotate(s["k"][:used], s["k_scale"], cos, sin)
    s["v_cache"].flatten(0, 1)[slot] = s["v"][:used]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    """All requests at once, padded to the longest, in 32 bits."""
    case, q = s["case"], s["q"]
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    tables, context, new = s["tables"], s["context"].long(), s["new"].long()
    requests, used, most = case["requests"], s["used"], s["most_new"]
    request, place, _, _ = _rows_of(s)
    request, place = request[:used], place[:used]
    rows = torch.zeros(requests, most, heads, dim, device=DEVICE)
    rows[request, place] = q[:used].float()
    rows = rows.view(requests, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(
        requests * kv_heads, -1, dim)
    length = tables.shape[1] * page
    pages = tables.long().clamp(min=0)
    keys = s["k_cache"][pages].view(requests, length, kv_heads, dim).permute(0, 2, 3, 1).float()
    scores = torch.bmm(rows, keys.reshape(requests * kv_heads, dim, length)) * dim ** -0.5
    del keys
    key = torch.arange(length, device=DEVICE)
    own_key = context[:, None] + torch.arange(most, device=DEVICE)[None, :]  # [requests, most]
    seen = key <= own_key[..., None]
    if case["window"]:
        seen &= key > own_key[..., None] - case["window"]
    scores = scores.view(requests, kv_heads, most, heads // kv_heads, length)
    scores.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    weights = torch.softmax(scores, dim=-1).view(requests * kv_heads, -1, length)
    del scores
    # what lies behind a request's last key is no value of it
    values = s["v_cache"][pages].view(requests, length, kv_heads, dim).float()
    values = values.masked_fill(~(key < (context + new)[:, None])[..., None, None], 0)
    values = values.permute(0, 2, 1, 3).reshape(requests * kv_heads, length, dim)
    found = torch.bmm(weights, values).view(requests, kv_heads, most, heads // kv_heads, dim)
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device=DEVICE)
    out[:used] = found.permute(0, 2, 1, 3, 4).reshape(requests, most, heads, dim)[request, place].to(torch.bfloat16)
    return out


def _plain_product(s):
    case, codes = s["case"], s["codes"]
    k, n, group = case["k"], case["n"], case["group"]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float()[:, None, :]
    w = ((codes.float().view(k // group, group, n) - zeros) * s["scales"].float()[:, None, :]).view(k, n)
    y = torch.matmul(s["x"].float(), w)
    if case["epilogue"] == "swiglu":
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    elif s["extra"] is not None:
        y = y + s["extra"].float()
    return y.to(torch.bfloat16)


def run(state):
    if own:
        return _own_pass(state)
    kind = state["case"]["kind"]
    if kind == "plan":
        return _plain_plan(state)
    if kind == "write":
        return _plain_write(state)
    if kind == "attention":
        return _plain_attention(state)
    return _plain_product(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    if case["kind"] == "int4":
        m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
        out = n // 2 if case["epilogue"] == "swiglu" else n
        extra = {"residual_add": 2 * m * n, "bias_add": 2 * n}.get(case["epilogue"], 0)
        weight = k * n / 2 + groups * n * (2.5 if case["zeros"] else 2)
        return {"bytes": weight + 2 * m * (k + out) + extra, "flops": 2 * m * k * n}
    context, new = (x.double() for x in _lengths(case))
    tokens, requests, page = float(new.sum()), case["requests"], case["page"]
    if case["kind"] == "plan":
        pages = float((torch.ceil((context + new) / page) - torch.ceil(context / page)).sum())
        return {"bytes": 16 * requests + 8 * pages + 12 * tokens, "flops": 8 * requests + 4 * tokens}
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["kind"] == "write":
        # heads once in and once out, two table rows and a slot a token
        return {"bytes": tokens * (4 * q + 8 * kv + 2 * case["dim"] + 12), "flops": tokens * 8 * (q + kv)}
    length = context + new
    # the keys a request's rows see in all: each row its own and those before it
    pairs = new * context + new * (new + 1) / 2
    if case["window"]:
        w = float(case["window"])
        ramp = (torch.minimum(length, torch.tensor(w)) - torch.minimum(context, torch.tensor(w)))  # rows not yet full
        low = torch.minimum(context, torch.tensor(w))
        pairs = ramp * low + ramp * (ramp + 1) / 2 + (new - ramp) * w
        length = torch.minimum(length, new + w - 1)
    return {"bytes": float(4 * tokens * q + (4 * kv + 4 / page) * length.sum()),
            "flops": float(4 * q * pairs.sum())}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    if case["kind"] == "int4":
        s = _product_inputs(case, seed)
        group, n = case["group"], case["n"]
        y = torch.zeros(case["m"], n, dtype=torch.float64, device=DEVICE)
        step = max(1, 4096 // group)  # groups at a time
        for g in range(0, case["k"] // group, step):
            part = slice(g * group, (g + step) * group)
            scale = s["scales"][g:g + step].double().repeat_interleave(group, 0)
            zero = 8 if s["zeros"] is None else s["zeros"][g:g + step].double().repeat_interleave(group, 0)
            y += s["x"][:, part].double() @ ((s["codes"][part].double() - zero) * scale)
        if case["epilogue"] == "swiglu":
            return torch.sigmoid(y[:, :n // 2]) * y[:, :n // 2] * y[:, n // 2:]
        return y if s["extra"] is None else y + s["extra"].double()
    s = _serve_inputs(case, seed)
    context, new = _lengths(case)
    page, dim, row = case["page"], case["dim"], 0
    if case["kind"] == "write":
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()

        def heads(x, scale, at):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + EPS) * scale.double()
            cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
            first, second = x[..., :dim // 2], x[..., dim // 2:]
            return torch.cat((first * cos - second * sin, first * sin + second * cos), -1)

        for b, (c, w) in enumerate(zip(context.tolist(), new.tolist())):
            at = torch.arange(c, c + w, device=DEVICE)
            pages, part = s["tables"][b].long()[at // page], slice(row, row + w)
            q[part] = heads(s["q"][part], s["q_scale"], at)
            k_cache[pages, at % page] = heads(s["k"][part], s["k_scale"], at)
            v_cache[pages, at % page] = s["v"][part].double()
            row += w
        return [q, k_cache, v_cache]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    ratio = case["heads"] // case["kv_heads"]
    for b, (c, w) in enumerate(zip(context.tolist(), new.tolist())):
        at = torch.arange(c + w, device=DEVICE)
        pages = s["tables"][b].long()[at // page]
        mine = at[c:, None]
        hidden = at[None, :] > mine
        if case["window"]:
            hidden = hidden | (at[None, :] <= mine - case["window"])
        for h in range(case["kv_heads"]):
            keys, values = (x[pages, at % page, h].double() for x in (s["k_cache"], s["v_cache"]))
            for j in range(h * ratio, (h + 1) * ratio):
                score = (s["q"][row:row + w, j].double() @ keys.t() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                score = torch.exp(score - score.amax(-1, keepdim=True))
                out[row:row + w, j] = (score @ values) / score.sum(-1, keepdim=True)
        row += w
    return out
