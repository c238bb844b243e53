"""The paged serving operators on the GPU: the plan against a loop over requests, the
write and the attention against their definitions in 64 bits, and the three together
as a serving step runs them."""

import math

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def expected_plan(context, new, tables, page, num_pages, tokens, free, max_new, max_context):
    """The plan as its description says, one request after another."""
    tables = [list(row) for row in tables]
    starts, status, rows, used, demand, needed = [0], [], [], 0, 0, 0
    positions, slots = [-1] * tokens, [-1] * tokens
    for b, (c, n) in enumerate(zip(context, new)):
        start = starts[-1]
        length = min(max(n, 0), tokens + 1)
        starts.append(start + length)
        why = smx.PAGED_OK
        if c < 0 or n < 0 or n > max_new or c + n > max_context:
            why = smx.PAGED_BAD_LENGTH
        elif n and start + n > tokens:
            why = smx.PAGED_OUT_OF_ROWS
        elif n and c % page and not 0 <= tables[b][c // page] < num_pages:
            why = smx.PAGED_BAD_PAGE
        elif n and free is not None:
            held, need = -(-c // page), -(-(c + n) // page) - -(-c // page)
            demand += need
            if need and demand > len(free):
                why = smx.PAGED_OUT_OF_PAGES
            elif need:
                tables[b][held:held + need] = free[demand - need:demand]
                used = demand
        if why == smx.PAGED_OK:
            needed = demand
        status.append(why)
        rows.append(n if why == smx.PAGED_OK else 0)
        for i in range(rows[-1]):
            positions[start + i] = c + i
            entry = tables[b][(c + i) // page]
            if 0 <= entry < num_pages:
                slots[start + i] = entry * page + (c + i) % page
    return starts, status, rows, positions, slots, used, needed, tables


def check_plan(context, new, tables, page, num_pages, tokens, free, max_new=None, max_context=None):
    width = len(tables[0])
    on_gpu = i32(tables)
    plan = smx.paged_plan(i32(context), i32(new), on_gpu, page_size=page, num_pages=num_pages, tokens=tokens,
                          free_pages=None if free is None else i32(free), max_new=max_new, max_context=max_context)
    want = expected_plan(context, new, tables, page, num_pages, tokens, free,
                         tokens if max_new is None else max_new, width * page if max_context is None else max_context)
    got = (plan.starts, plan.status, plan.rows, plan.positions, plan.slots, int(plan.pages_used), int(plan.pages_needed), on_gpu)
    for name, g, w in zip(("starts", "status", "rows", "positions", "slots", "pages_used", "pages_needed", "tables"), got, want):
        g = g.tolist() if isinstance(g, torch.Tensor) else g
        assert g == w, name
    assert plan.context.tolist() == [c if s == 0 else 0 for c, s in zip(context, want[1])]
    assert (plan.slots.dtype, plan.positions.dtype) == (torch.int64, torch.int32)
    return plan


def tables_of(context, width, page, order):
    """Block tables of the contexts' pages, and the pages left over."""
    order, tables = list(order), []
    for c in context:
        held = -(-c // page)
        tables.append([order.pop(0) for _ in range(held)] + [-1] * (width - held))
    return tables, order


@pytest.mark.parametrize("context,new,page,tokens", [
    ([0], [1], 16, 1), ([15], [1], 16, 16), ([16], [1], 16, 3), ([7, 0, 31], [9, 0, 33], 8, 48),
    ([0, 0, 5], [0, 0, 0], 8, 4), ([100, 1, 64, 0], [28, 64, 1, 200], 64, 300),
])
def test_plan(context, new, page, tokens):
    width = max(-(-(c + n) // page) for c, n in zip(context, new)) + 1
    generator = torch.Generator().manual_seed(1)
    pages = sum(-(-(c + n) // page) for c, n in zip(context, new)) + 3
    order = torch.randperm(pages, generator=generator).tolist()
    tables, free = tables_of(context, width, page, order)
    check_plan(context, new, tables, page, pages, tokens, free)


def test_plan_of_many_requests():
    """More requests than threads, more tokens than one workgroup lays out."""
    generator = torch.Generator().manual_seed(2)
    requests, page = 2500, 8
    context = torch.randint(0, 90, (requests,), generator=generator).tolist()
    new = torch.randint(0, 5, (requests,), generator=generator).tolist()
    width = 13
    order = torch.randperm(40000, generator=generator).tolist()
    tables, free = tables_of(context, width, page, order)
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(context, new) if n)
    check_plan(context, new, tables, page, 40000, sum(new) + 7, free)
    plan = check_plan(context, new, tables, page, 40000, sum(new) + 7, free[:need // 2])
    assert (plan.status == smx.PAGED_OUT_OF_PAGES).any()


def test_plan_refuses_requests_one_by_one():
    """Lengths, rows, pages and tables that a step cannot take leave the other requests as they are."""
    page, width, pages = 8, 4, 40
    context = [3, -1, 5, 30, 8, 8, 0, 16, 9]
    new = [1, 2, -4, 3, 9, 2, 1, 8, 1]
    tables = [[b * 4 + i for i in range(4)] for b in range(9)]
    tables[0][0], tables[8][1] = 40, -3  # no pages of the cache
    check_plan(context, new, tables, page, pages, 26, [36, 37, 38, 39], max_new=8)
    check_plan(context, new, tables, page, pages, 26, [36], max_new=8)
    check_plan(context, new, tables, page, pages, 12, [], max_new=8)  # out of rows, no free page
    check_plan(context, new, tables, page, pages, 26, None, max_new=9, max_context=20)
    check_plan([0, 0], [2**31 - 1, 3], [[0], [1]], page, pages, 5, [2, 3])  # lengths whose sum passes 32 bits
    check_plan([2**31 - 1, 0], [1, 3], [[0], [1]], page, pages, 5, [2, 3])
    # pages of the list that the cache does not have: no slots, the request keeps its rows
    check_plan([0, 8], [9, 1], [[-1, -1], [5, -1]], page, pages, 10, [41, 7, -2])


def make_step(context, new, *, page, kv_heads, dim, pad=0, seed=0, layout="pages", spare=3, width=None):
    """A cache with NaN wherever no request holds a token, its plan, and its keys and
    values in 64 bits by request."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = sum(-(-(c + n) // page) for c, n in zip(context, new)) + spare
    if layout == "pages":
        k, v = (torch.full((pages, page, kv_heads, dim), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    elif layout == "heads":  # heads outside the page's tokens
        k, v = (torch.full((pages, kv_heads, page, dim), math.nan, dtype=torch.bfloat16, device=DEV).transpose(1, 2)
                for _ in range(2))
    else:  # one tensor for both, padded heads
        both = torch.full((pages, 2, page, kv_heads, dim + 8), math.nan, dtype=torch.bfloat16, device=DEV)
        k, v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    width = width or max(1, max(-(-(c + n) // page) for c, n in zip(context, new)))
    tables, _ = tables_of([c + n for c, n in zip(context, new)], width, page, order)
    keys, values = [], []
    for b, (c, n) in enumerate(zip(context, new)):
        at = torch.arange(c + n, device=DEV)
        rows, offsets = i32(tables[b]).long()[at // page], at % page
        for cache, kept in ((k, keys), (v, values)):
            x = torch.randn(c + n, kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16)
            cache[rows, offsets] = x
            kept.append(x.double())
    plan = smx.paged_plan(i32(context), i32(new), i32(tables), page_size=page, num_pages=pages,
                          tokens=max(1, sum(new) + pad))
    return plan, k, v, keys, values, g


def attend64(q, keys, values, context, new, window, scale=None, unseen=()):
    """(result, sum of weights times |v|) of every row of the requests."""
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    row, heads = 0, q.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for b, (c, n) in enumerate(zip(context, new)):
        key, own = torch.arange(c + n, device=DEV), torch.arange(c, c + n, device=DEV)[:, None]
        hidden = key > own
        if window:
            hidden = hidden | (key <= own - window)
        for bb, j in unseen:
            if bb == b:
                hidden = hidden | (key == j)
        for h in range(heads if n else 0):
            kv = h // (heads // keys[b].shape[1])
            s = (q[row:row + n, h].double() @ keys[b][:, kv].T * scale).masked_fill(hidden, -math.inf)
            w = torch.softmax(s, dim=-1).nan_to_num(0.0)  # a row that sees nothing is zero
            out[row:row + n, h], size[row:row + n, h] = w @ values[b][:, kv], w @ values[b][:, kv].abs()
        row += n
    return out, size


def check_attention(got, want, size):
    """The weights are rounded to bf16 (2^-8 of each term) and the result once more; the FP32
    scores (128 products of a few units) move a weight by under 1e-3 of it."""
    assert got.isfinite().all()
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * size + 1e-30).all()


ATTENTION = [
    # context, new, page, heads, kv_heads, dim, window, layout
    ([0], [1], 8, 8, 8, 128, None, "pages"),
    ([63], [1], 16, 8, 2, 128, None, "pages"),
    ([64], [1], 64, 8, 2, 64, None, "pages"),
    ([0, 0], [65, 1], 16, 16, 2, 128, None, "pages"),
    ([5, 0, 200, 17], [0, 3, 1, 40], 8, 14, 2, 128, None, "heads"),
    ([31, 1000, 0], [1, 1, 1], 32, 40, 8, 64, None, "one"),
    ([700, 129], [300, 257], 16, 8, 1, 128, None, "pages"),
    ([3, 500], [130, 131], 128, 3, 3, 64, None, "heads"),
    ([90, 33], [5, 64], 16, 128, 1, 128, None, "pages"),  # every head of a token in a tile of its own
    ([400, 0], [70, 90], 16, 8, 2, 128, 1, "pages"),  # only itself
    ([400, 0, 63], [70, 90, 3], 16, 8, 2, 128, 64, "pages"),
    ([2000, 10], [33, 300], 64, 20, 4, 64, 100, "one"),
    ([9000, 3], [1, 1], 16, 16, 2, 128, None, "pages"),  # split and joined
    ([1500, 30, 0, 800], [600, 1, 1, 0], 16, 16, 8, 128, 5000, "pages"),
]


@pytest.mark.parametrize("context,new,page,heads,kv_heads,dim,window,layout", ATTENTION)
def test_attention(context, new, page, heads, kv_heads, dim, window, layout):
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, pad=5, layout=layout)
    q = (1.5 * torch.randn(plan.tokens, heads, dim, device=DEV, generator=g)).to(torch.bfloat16)
    q[sum(new):] = math.nan  # rows behind the last request
    want, size = attend64(q, keys, values, context, new, window)
    got = smx.paged_attention(q, k, v, plan, window=window)
    check_attention(got, want, size)
    assert not got[sum(new):].any()
    # the same bits again, on strided query heads, and with a bound on the step's new tokens
    wide = torch.cat((q, q), dim=1)
    assert torch.equal(smx.paged_attention(wide[:, heads:], k, v, plan, window=window), got)


@pytest.mark.parametrize("new", [[1] * 5, [3, 1, 2, 4, 1]])
def test_attention_of_a_bounded_step(new):
    """A decode step, its plan told how many tokens a request appends at most."""
    context, heads, kv_heads, dim, page = [0, 40, 1300, 7, 259], 64, 8, 128, 16
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, pad=3)
    bounded = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                             tokens=plan.tokens, max_new=max(new))
    q = torch.randn(plan.tokens, heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    for window in (None, 33):
        want, size = attend64(q, keys, values, context, new, window)
        check_attention(smx.paged_attention(q, k, v, bounded, window=window), want, size)
        check_attention(smx.paged_attention(q, k, v, plan, window=window), want, size)


@pytest.mark.parametrize("max_new", [None, 4])
def test_attention_leaves_out_pages_that_are_not_in_the_cache(max_new):
    """Entries behind or before the cache's pages: their keys are not seen, and rows that see none are zero."""
    context, new, page = [40, 2, 120], [2, 3, 1], 8
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=2, dim=128, pad=2)
    tables = plan.block_tables
    tables[0, 1], tables[0, 5], tables[1, 0], tables[2, 14] = -1, plan.num_pages, 2**31 - 1, -2**31
    unseen = [(0, j) for j in range(8, 16)] + [(0, j) for j in range(40, 48)] + [(1, j) for j in range(8)]
    unseen += [(2, j) for j in range(112, 120)]
    if max_new is not None:
        # admitted by an earlier plan; the tables change afterwards
        kept = plan.block_tables.clone()
        plan.block_tables.copy_(i32([[0] * tables.shape[1]] * 3))
        bounded = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                                 tokens=plan.tokens, max_new=max_new)
        plan.block_tables.copy_(kept)
        plan = bounded
    q = torch.randn(plan.tokens, 8, 128, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, None, unseen=unseen)
    got = smx.paged_attention(q, k, v, plan)
    check_attention(got, want, size)
    assert not got[2:5].any()


@pytest.mark.parametrize("new_high,max_new", [(1, 1), (3, 4), (3, None)])
@pytest.mark.parametrize("window", [None, 40])
def test_attention_of_many_requests(new_high, max_new, window):
    """More requests than a workgroup looks at in one round, some of them idle."""
    generator = torch.Generator().manual_seed(7)
    requests = 700
    context = torch.randint(0, 150, (requests,), generator=generator).tolist()
    new = torch.randint(0, new_high + 1, (requests,), generator=generator).tolist()
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=1, dim=64, pad=1)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, 4, 64, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, window)
    check_attention(smx.paged_attention(q, k, v, plan, window=window), want, size)


@pytest.mark.parametrize("heads,kv_heads,max_new", [(64, 8, 1), (8, 2, 4), (16, 2, 16)])
def test_attention_gives_the_same_bits_again(heads, kv_heads, max_new):
    """Many spans that begin and end within requests, their keys from memory: nothing is used before it has arrived."""
    context = [(b * 997) % 4000 + 1 for b in range(48)]
    new = [1 + b % max_new for b in range(48)]
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=kv_heads, dim=128)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, heads, 128, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, None)
    got = smx.paged_attention(q, k, v, plan)
    check_attention(got, want, size)
    other = torch.empty(1 << 28, device=DEV)
    for _ in range(12):
        other.zero_()  # leaves nothing of the cache in the caches
        assert torch.equal(smx.paged_attention(q, k, v, plan), got)


@pytest.mark.parametrize("heads,kv_heads,max_new", [(8, 8, 32), (32, 1, 1), (6, 2, 10), (64, 2, 1)])
@pytest.mark.parametrize("window", [None, 1, 2**31 - 1])
def test_attention_of_few_rows(heads, kv_heads, max_new, window):
    """Steps whose rows fill a tile of 32, nearly fill it or hold one token in it."""
    context, new = [600, 0, 33, 64], [max_new, max_new, 1, max(1, max_new // 2)]
    plan, k, v, keys, values, g = make_step(context, new, page=8, kv_heads=kv_heads, dim=128, pad=2)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=8, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, heads, 128, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, window)
    check_attention(smx.paged_attention(q, k, v, plan, window=window), want, size)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,new,max_new,window", [
    ([40, 0, 300], [1, 1, 1], 1, 16),  # behind the window, in the step's first keys
    ([30, 5, 200], [4, 3, 4], 4, None), ([30, 5, 200], [4, 3, 4], 4, 8),  # tokens of the step that come later
    ([0, 100], [150, 70], None, None), ([90, 700], [150, 70], None, 33),
])
def test_attention_of_rows_that_do_not_see_an_infinity_or_nan(dim, context, new, max_new, window):
    """Infinities and NaN among a request's values, and NaN among its keys, reach the rows that see them and no
    others."""
    page, kv_heads, heads = 8, 2, 4
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    for b, (c, n) in enumerate(zip(context, new)):
        odd = [(0, 0, math.inf), (max(0, c - 9), 3, math.nan), (c + n // 2, 5, -math.inf), (c + n - 1, 40, math.inf),
               (c + n - 1, 5, math.inf), (c + n - 1, 41, -math.inf), (c, 63, math.nan)]
        for at, column, value in odd:
            page_at = plan.block_tables[b, at // page]
            v[page_at, at % page, 1, column] = value
            values[b][at, 1, column] = value
        k[plan.block_tables[b, (c + n - 1) // page], (c + n - 1) % page, 0, 7] = math.nan
        keys[b][c + n - 1, 0, 7] = math.nan
    finite = [x.masked_fill(~x.isfinite(), 0.0) for x in values]
    got = smx.paged_attention(q, k, v, plan, window=window).double()
    want, size = attend64(q, [x.nan_to_num(0.0) for x in keys], finite, context, new, window)
    row = 0
    for b, (c, n) in enumerate(zip(context, new)):
        key, own = torch.arange(c + n, device=DEV), torch.arange(c, c + n, device=DEV)[:, None]
        sees = ((key <= own) & (key > own - (window or 1 << 30))).double()
        value = values[b][:, 1]
        up, down = (sees @ ((value == way) | value.isnan()).double() > 0 for way in (math.inf, -math.inf))
        part = want[row:row + n, 2:]  # the second key/value head's query heads
        part[up[:, None].expand_as(part)] = math.inf
        part[down[:, None].expand_as(part)] = -math.inf
        part[(up & down)[:, None].expand_as(part)] = math.nan
        want[row + n - 1, :2] = math.nan  # the last row alone sees the key
        row += n
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == math.inf, want == math.inf) and torch.equal(got == -math.inf, want == -math.inf)
    here = want.isfinite()
    check_attention(got[here], want[here], size[here])


def test_one_page_one_head_views():
    """Dimensions of one, whose strides mean nothing."""
    plan, k, v, keys, values, g = make_step([3], [2], page=8, kv_heads=1, dim=64, spare=0)
    q = torch.randn(2, 1, 64, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, [3], [2], None)
    odd = [x.as_strided((1, 8, 1, 64), s) for x, s in ((k, (0, 64, 3, 1)), (v, (7, 64, 512, 1)))]
    check_attention(smx.paged_attention(q.as_strided((2, 1, 64), (64, 5, 1)), *odd, plan), want, size)


def test_attention_scale_and_out():
    context, new = [70, 12], [9, 1]
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=2, dim=64, pad=6)
    q = torch.randn(plan.tokens, 4, 64, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, None, scale=0.5)
    out = torch.full((plan.tokens, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    assert smx.paged_attention(q, k, v, plan, scale=0.5, out=out) is out
    check_attention(out[:10], want[:10], size[:10])
    assert (out[10:] == 7).all()  # rows behind the last request stay


@pytest.mark.parametrize("max_new", [None, 2])
def test_attention_in_place_of_the_queries(max_new):
    """Each row is read before it is written, also those of requests that several workgroups share."""
    context, new = [5000, 12, 700], [2, 1, 2]
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=2, dim=128)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, 16, 128, device=DEV, generator=g).to(torch.bfloat16)
    want = smx.paged_attention(q, k, v, plan)
    assert smx.paged_attention(q, k, v, plan, out=q) is q
    assert torch.equal(q, want)


def test_attention_of_a_long_prompt():
    """100,000 rows of one request, whose tiles' counts pass 16 bits, against sampled rows."""
    new, page, heads = 100_000, 64, 2
    plan, k, v, keys, values, g = make_step([0], [new], page=page, kv_heads=1, dim=64)
    q = torch.randn(new, heads, 64, device=DEV, generator=g).to(torch.bfloat16)
    got = smx.paged_attention(q, k, v, plan)
    for row in (0, 1, 63, 64, 4095, 31337, 65535, 65536, new - 2, new - 1):
        want, size = attend64(q[row:row + 1], [keys[0][:row + 1]], [values[0][:row + 1]], [row], [1], None)
        check_attention(got[row:row + 1], want, size)
    assert got.isfinite().all()


def test_attention_of_requests_that_are_not_admitted():
    """Their rows are zero, the others' as if alone."""
    plan, k, v, keys, values, g = make_step([20, 30, 4], [3, 5, 2], page=8, kv_heads=2, dim=64, pad=1)
    q = torch.randn(plan.tokens, 2, 64, device=DEV, generator=g).to(torch.bfloat16)
    got = smx.paged_attention(q, k, v, plan)
    less = smx.paged_plan(i32([20, 30, 4]), i32([3, 5, 2]), plan.block_tables, page_size=8, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=4)
    assert less.status.tolist() == [smx.PAGED_OK, smx.PAGED_BAD_LENGTH, smx.PAGED_OK]
    rest = smx.paged_attention(q, k, v, less)
    assert not rest[3:8].any() and torch.equal(rest[:3], got[:3]) and torch.equal(rest[8:], got[8:])


def test_attention_past_32_bit_offsets():
    """Pages whose offsets pass 2^31 elements and 2^32 bytes."""
    pages, page, kv_heads, dim = 140000, 16, 8, 128
    both = torch.empty(pages, 2, page, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
    k, v = both[:, 0], both[:, 1]
    context, new = [100, 40], [20, 1]
    tables = [[139990 + i if i % 2 else i for i in range(8)], [70000 + i for i in range(3)] + [0] * 5]
    plan = smx.paged_plan(i32(context), i32(new), i32(tables), page_size=page, num_pages=pages, tokens=21)
    g = torch.Generator(device=DEV).manual_seed(3)
    keys, values = [], []
    for b, (c, n) in enumerate(zip(context, new)):
        at = torch.arange(c + n, device=DEV)
        for cache, kept in ((k, keys), (v, values)):
            x = torch.randn(c + n, kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16)
            cache[i32(tables[b]).long()[at // page], at % page] = x
            kept.append(x.double())
    fresh = [[torch.cat([kept[b][c:c + n] for b, (c, n) in enumerate(zip(context, new))]).to(torch.bfloat16)]
             for kept in (keys, values)]
    smx.paged_write(fresh[0][0], fresh[1][0], k, v, plan)
    q = torch.randn(21, 16, dim, device=DEV, generator=g).to(torch.bfloat16)
    want, size = attend64(q, keys, values, context, new, None)
    check_attention(smx.paged_attention(q, k, v, plan), want, size)


def rotate64(x, scale, cos, sin, eps):
    x = x.double()
    if scale is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * scale.double()
    if cos is None:
        return x
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos.double()[:, None, :half], sin.double()[:, None, :half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


@pytest.mark.parametrize("dim,heads,kv_heads,layout", [(128, 16, 2, "pages"), (64, 5, 5, "heads"), (128, 1, 1, "one")])
@pytest.mark.parametrize("norm,rope,dtype", [(True, True, torch.bfloat16), (True, False, torch.float32),
                                             (False, True, torch.float32), (False, False, torch.bfloat16)])
def test_write(dim, heads, kv_heads, layout, norm, rope, dtype):
    context, new, page = [5, 0, 30], [4, 0, 19], 16
    plan, k_cache, v_cache, *_, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, pad=4, layout=layout)
    qkv = torch.randn(plan.tokens, heads + 2 * kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), dim=1)
    before = [k_cache.clone(), v_cache.clone()]
    options = {}
    if norm:
        options.update({f"{x}_scale": torch.randn(dim, device=DEV, generator=g).to(dtype) for x in "qk"})
    if rope:
        angle = torch.rand(plan.max_context, dim // 2, device=DEV, generator=g) * 100
        if dtype == torch.float32:
            angle = torch.cat((angle, angle), dim=-1)  # tables of whole heads
        options.update(rope_cos=torch.cos(angle).to(dtype), rope_sin=torch.sin(angle).to(dtype))
    out = smx.paged_write(k, v, k_cache, v_cache, plan, q=q, eps=1e-5, **options)
    used = sum(new)
    at = plan.positions[:used].long()
    cos, sin = (options[x][at] if rope else None for x in ("rope_cos", "rope_sin"))
    slots = plan.slots[:used]
    for got, x, scale in ((out[:used], q, "q_scale"), (k_cache[slots // page, slots % page], k, "k_scale")):
        want = rotate64(x[:used], options.get(scale), cos, sin, 1e-5)
        # one rounding, and FP32 rounding of the terms (their sum may cancel)
        bound = 2.0 ** -8 * want.abs() + 2.0 ** -18 * rotate64(x[:used], options.get(scale), None, None, 1e-5).abs().amax(-1, keepdim=True)
        assert ((got.double() - want).abs() <= bound + 1e-30).all()
    assert torch.equal(v_cache[slots // page, slots % page], v[:used])
    assert not out[used:].any()
    # nothing but the step's slots has changed
    for cache, old in zip((k_cache, v_cache), before):
        cache[slots // page, slots % page] = old[slots // page, slots % page]
        assert torch.equal(cache.isnan(), old.isnan())
        assert torch.equal(cache.nan_to_num(), old.nan_to_num())


def test_write_of_keys_alone():
    plan, k_cache, v_cache, *_, g = make_step([3], [9], page=8, kv_heads=2, dim=128)
    k, v = (torch.randn(9, 2, 128, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    assert smx.paged_write(k, v, k_cache, v_cache, plan) is None
    assert torch.equal(k_cache[plan.slots // 8, plan.slots % 8], k)
    assert torch.equal(v_cache[plan.slots // 8, plan.slots % 8], v)


def run_step(s):
    plan = smx.paged_plan(s["context"], s["new"], s["tables"], page_size=16, num_pages=s["k_cache"].shape[0],
                          tokens=s["q"].shape[0], free_pages=s["free"], max_new=s["max_new"])
    q = smx.paged_write(s["k"], s["v"], s["k_cache"], s["v_cache"], plan, q=s["q"], rope_cos=s["cos"],
                        rope_sin=s["sin"], q_scale=s["scale"], k_scale=s["scale"])
    return smx.paged_attention(q, s["k_cache"], s["v_cache"], plan), plan


def step_state(max_new=64):
    g = torch.Generator(device=DEV).manual_seed(4)
    s = {"k_cache": torch.zeros(64, 16, 2, 128, dtype=torch.bfloat16, device=DEV), "max_new": max_new}
    s["v_cache"] = torch.zeros_like(s["k_cache"])
    s["context"], s["new"] = i32([0, 0, 0]), i32([20, 1, 7])
    s["tables"] = i32([[-1] * 16] * 3)
    s["free"] = torch.randperm(64, device=DEV, generator=g).to(torch.int32)
    s["q"] = torch.randn(32, 8, 128, device=DEV, generator=g).to(torch.bfloat16)
    s["k"], s["v"] = (torch.randn(32, 2, 128, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    angle = torch.rand(256, 64, device=DEV, generator=g) * 50
    s["cos"], s["sin"] = torch.cos(angle).to(torch.bfloat16), torch.sin(angle).to(torch.bfloat16)
    s["scale"] = (1 + 0.1 * torch.randn(128, device=DEV, generator=g)).to(torch.bfloat16)
    return s, g


def advance(s, plan, g, new):
    """The lengths, the free list and the heads of the next step, in place."""
    s["context"].add_(plan.rows)
    s["free"].copy_(torch.roll(s["free"], -int(plan.pages_used)))
    s["new"].copy_(i32(new))
    for x in ("q", "k", "v"):
        s[x].copy_(torch.randn(s[x].shape, device=DEV, generator=g))


def test_steps_build_on_each_other():
    """A prompt in pieces with decoding beside it gives what whole sequences give: every
    step's rows against the 64-bit attention over all keys stored so far."""
    s, g = step_state()
    keys, values = [[] for _ in range(3)], [[] for _ in range(3)]
    for new in ([20, 1, 7], [5, 0, 20], [1, 1, 1], [30, 1, 0]):
        s["new"].copy_(i32(new))
        context = s["context"].tolist()
        out, plan = run_step(s)
        assert plan.status.tolist() == [0, 0, 0]
        row, q64 = 0, torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(new):
            at, part = torch.arange(context[b], context[b] + n, device=DEV), slice(row, row + n)
            rot = [rotate64(s[x][part], s["scale"], s["cos"][at], s["sin"][at], 1e-6).to(torch.bfloat16) for x in "qk"]
            q64[part] = rot[0].double()
            keys[b].append(rot[1].double())
            values[b].append(s["v"][part].double())
            row += n
        want, size = attend64(q64, [torch.cat(x) for x in keys], [torch.cat(x) for x in values], context, new, None)
        # the heads themselves may round the other way: 2^-8 of the scores' terms, some 16 units at most
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 0.15) * size + 1e-30).all()
        assert (out.double() - want).norm() <= 1e-2 * want.norm()
        advance(s, plan, g, new)


@pytest.mark.parametrize("max_new", [64, 1])
def test_step_in_a_graph(max_new):
    """Captured once and replayed with other lengths, pages and heads: each replay gives
    the eager step's bits; so do two graphs replayed in turn."""
    first = [20, 1, 7] if max_new > 1 else [1, 1, 1]
    later = ([1, 1, 1], [0, 9, 2], [31, 0, 1]) if max_new > 1 else ([1, 1, 1], [0, 1, 1], [1, 0, 0])
    s, g = step_state(max_new)
    s["new"].copy_(i32(first))
    run_step(s)  # loads kernels outside the capture
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = run_step(s)
        graphs.append((graph, captured))
    for i, new in enumerate(later):
        _, plan = run_step(s)
        advance(s, plan, g, new)
        saved = {x: s[x].clone() for x in ("tables", "k_cache", "v_cache")}
        want, _ = run_step(s)
        after = {x: s[x].clone() for x in saved}
        for graph, captured in graphs:
            for x, old in saved.items():
                s[x].copy_(old)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(captured[0], want)
            assert all(torch.equal(s[x], after[x]) for x in after)


def test_calls_on_two_streams():
    """Two calls at once, each with its own workspace, give what they give alone."""
    plan, k, v, *_, g = make_step([3000, 50], [40, 1], page=16, kv_heads=2, dim=128)
    q = [torch.randn(plan.tokens, 8, 128, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2)]
    alone = [smx.paged_attention(x, k, v, plan) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, x in zip(streams, q):
            with torch.cuda.stream(stream):
                got.append(smx.paged_attention(x, k, v, plan))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))


def test_refusals():
    plan, k, v, *_, g = make_step([9], [4], page=8, kv_heads=2, dim=128)
    q = torch.randn(4, 8, 128, device=DEV, generator=g).to(torch.bfloat16)
    good = dict(q=q, k_cache=k, v_cache=v, plan=plan)
    for change, message in (
            ({"q": q[:3]}, "shape"), ({"q": q.float()}, "bf16"), ({"q": q[:, :7]}, "query heads"),
            ({"q": q[..., :64]}, "shape"), ({"k_cache": k[:1]}, "same shape"),
            ({"k_cache": k[:2], "v_cache": v[:2]}, "pages"), ({"scale": 0.0}, "scale"), ({"scale": math.inf}, "scale"),
            ({"window": 0}, "window"), ({"window": -3}, "window"), ({"out": q.float()}, "bf16"),
            ({"out": torch.empty(4, 8, 130, dtype=torch.bfloat16, device=DEV)[..., 1:129]}, "aligned"),
            ({"out": torch.empty(1, 8, 128, dtype=torch.bfloat16, device=DEV).expand(4, 8, 128)}, "on each other"),
            ({"q": q.cpu()}, "HIP device"), ({"q": q.clone().requires_grad_()}, "gradients")):
        with pytest.raises(ValueError, match=message):
            smx.paged_attention(**{**good, **change})
    cos = torch.zeros(plan.max_context, 64, device=DEV)
    for args, message in (
            ({"q_scale": cos[0].repeat(2)}, "without q"), ({"rope_cos": cos}, "go together"),
            ({"rope_cos": cos[1:], "rope_sin": cos[1:]}, "positions"),
            ({"rope_cos": cos[:, :32], "rope_sin": cos[:, :32]}, "values"),
            ({"rope_cos": cos, "rope_sin": cos.bfloat16()}, "both"), ({"k_scale": cos[0]}, "shape")):
        with pytest.raises(ValueError, match=message):
            smx.paged_write(q[:, :2], q[:, :2], k, v, plan, **args)
    with pytest.raises(ValueError, match="shape"):
        smx.paged_write(q, q[:, :2], k, v, plan)
    lens, tables = i32([1, 2]), i32([[0], [1]])
    good = dict(context_lens=lens, new_lens=lens, block_tables=tables, page_size=8, num_pages=4, tokens=5)
    for change, message in (
            ({"new_lens": lens.long()}, "int32"), ({"new_lens": lens[:1]}, "shape"), ({"block_tables": tables[:1]}, "block_tables"),
            ({"block_tables": tables.long()}, "block_tables"), ({"page_size": 12}, "power of two"), ({"page_size": 4}, "power of two"),
            ({"tokens": 0}, "tokens"), ({"num_pages": 0}, "cache"), ({"max_context": 9}, "max_context"),
            ({"free_pages": lens.long()}, "int32"), ({"max_new": -1}, "max_context")):
        with pytest.raises(ValueError, match=message):
            smx.paged_plan(**{**good, **change})
