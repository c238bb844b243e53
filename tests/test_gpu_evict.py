"""Eviction from the paged cache on the GPU against a loop over requests and heads: everything it leaves, bit by bit."""

import math

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_paged import i32
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def make_cache(context, *, page=16, kv_heads=2, dim=64, layout="pages", seed=0, spare=3, width=None):
    """A cache whose every value is its own (so that a row out of place shows), shuffled tables and received weights."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    held = [-(-max(c, 0) // page) for c in context]
    pages = sum(held) + spare
    if layout == "pages":
        k, v = (torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    elif layout == "heads":
        k, v = (torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2))
    else:
        both = torch.zeros(pages, 2, page, kv_heads, dim + 8, dtype=torch.bfloat16, device=DEV)
        k, v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
    for x in (k, v):
        x.copy_(torch.randn(x.shape, device=DEV, generator=g))
    weights = torch.randn(pages, kv_heads, page, device=DEV, generator=g).exp()
    order = torch.randperm(pages, device=DEV, generator=g).tolist()
    width = width or max(1, max(held))
    tables = [[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    return k, v, weights, i32(context), i32(tables)


def expected(k, v, weights, context, tables, keep, recent, max_context=None):
    """Request by request, head by head, on the CPU."""
    k, v, weights = (x.clone().cpu() for x in (k.contiguous(), v.contiguous(), weights))
    pages, page, kv_heads, _ = k.shape
    tables = tables.cpu()
    most = tables.shape[1] * page if max_context is None else max_context
    lens = []
    for b, n in enumerate(context):
        goal = keep[b] if isinstance(keep, list) else keep
        lens.append(n)
        if n <= goal or n > most or goal < 0:
            continue
        entries = tables[b, :(n - 1) // page + 1]
        if ((entries < 0) | (entries >= pages)).any():
            continue
        lens[-1] = goal
        at = torch.arange(n)
        of, slot = entries.long()[at // page], at % page
        last = min(recent, goal)
        need, old = goal - last, n - last
        for h in range(kv_heads):
            mine = weights[of, h, slot]
            ranked = mine[:old].nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf).double()
            ranked = ranked + mine[:old].isnan().double()  # (inf stays inf: a NaN comes first among them)
            best = sorted(range(old), key=lambda i: (not math.isnan(mine[i]), -ranked[i].item(), i))[:need]
            places = sorted(set(range(need)) - set(best))
            movers = sorted(i for i in best if i >= need)
            to = torch.tensor(places + list(range(need, goal)), dtype=torch.long)
            frm = torch.tensor(movers + list(range(old, n)), dtype=torch.long)
            for x in (k, v):
                x[of[to], slot[to], h] = x[of[frm], slot[frm], h]
            weights[of[to], h, slot[to]] = mine[frm]
    return k, v, weights, lens


def same(got, want):
    """Equal bits (NaN among them)."""
    kind = torch.int16 if got.dtype == torch.bfloat16 else torch.int32
    return torch.equal(got.contiguous().cpu().view(kind), want.contiguous().view(kind))


def check(cache, context, keep, recent, **kw):
    k, v, weights, lens, tables = cache
    want = expected(k, v, weights, context, tables, keep, recent, kw.get("max_context"))
    before = tables.clone()
    got = smx.paged_evict(k, v, weights, lens, tables, i32(keep) if isinstance(keep, list) else keep, recent=recent, **kw)
    assert got.dtype == torch.int32 and got.tolist() == want[3]
    assert lens.tolist() == context and torch.equal(tables, before)
    assert same(weights, want[2]), "weights"
    assert same(k, want[0]), "keys"
    assert same(v, want[1]), "values"


@pytest.mark.parametrize("context,keep,recent", [
    ([1], 0, 0), ([1], 1, 1), ([2], 1, 0), ([2], 1, 1), ([17], 16, 0), ([17], 16, 16), ([17], 16, 1000), ([100], 1, 0),
    ([100, 3, 0, 64, 65], 64, 10), ([300, 299, 260, 257, 256], 256, 200), ([500], 100, 100), ([500], 400, 150), ([500], 0, 7),
    ([1000, 40, 777], 333, 0), ([5000, 4097, 4096], 700, 33),
])
@pytest.mark.parametrize("page,kv_heads,dim,layout", [(16, 2, 64, "pages"), (8, 1, 128, "one"), (128, 3, 128, "heads")])
def test_evict(context, keep, recent, page, kv_heads, dim, layout):
    check(make_cache(context, page=page, kv_heads=kv_heads, dim=dim, layout=layout, seed=sum(context) + keep), context, keep, recent)


@pytest.mark.parametrize("recent", [0, 40, 2000])
def test_lengths_of_each_request(recent):
    context = [90, 500, 64, 2000, 31, 0, 1]
    check(make_cache(context, seed=1), context, [30, 499, 64, 1000, -1, 0, 0], recent)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "odd", "close", "ordered", "halves"])
def test_equal_and_odd_weights(kind):
    """Ties go to the lowest index; NaN before infinities; values that share all of their leading bits."""
    context = [3000, 700, 1500]
    cache = make_cache(context, seed=2)
    w = cache[2]
    g = torch.Generator(device=DEV).manual_seed(3)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_(torch.randint(0, 4, w.shape, device=DEV, generator=g))
    elif kind == "zeros":
        w.mul_(torch.rand(w.shape, device=DEV, generator=g) < 0.1)
        w.mul_(torch.where(torch.rand(w.shape, device=DEV, generator=g) < 0.5, -1.0, 1.0))  # -0 is 0
        w.abs_().mul_(torch.where(w == 0, -1.0, 1.0))
    elif kind == "odd":
        pick = torch.rand(w.shape, device=DEV, generator=g)
        w[pick < 0.3], w[pick < 0.2], w[pick < 0.1] = math.inf, math.nan, -math.inf
        w.mul_(torch.where(pick > 0.8, -1.0, 1.0))
        w[pick > 0.95] = -math.nan
    elif kind == "close":
        w.copy_((torch.full(w.shape, 1.0, device=DEV).view(torch.int32) + torch.randint(0, 5, w.shape, device=DEV, generator=g).int()).view(torch.float32))
    elif kind == "ordered":
        w.copy_(torch.arange(w.numel(), device=DEV).view(w.shape))
    else:  # one value above a crowd that needs a second look
        w.copy_(1 + torch.rand(w.shape, device=DEV, generator=g) * 2**-12)
        w.view(-1)[::997] = 1e30
    check(cache, context, 600, 50)


@pytest.mark.parametrize("context,keep,recent,page", [([40000], 9000, 300, 64), ([70001, 33000, 32768 + 16], 32768, 16, 16),
                                                      ([131000], 1000, 0, 128)])
def test_long_contexts(context, keep, recent, page):
    """More tokens than a workgroup's registers hold."""
    check(make_cache(context, kv_heads=1, page=page, seed=4), context, keep, recent)


@pytest.mark.parametrize("kind", ["any", "equal", "few", "zeros", "odd", "close", "halves", "rising", "falling"])
def test_long_contexts_in_parts(kind):
    """Several workgroups a head: weights that crowd at the edge, that are equal across parts, that rise or fall along a request (so
    that the first thousand say little about the others), next to short requests and those that stay."""
    context = [50000, 8192, 8193, 40, 0, 33000, 16384, 20000]
    cache = make_cache(context, page=32, seed=20)
    k, v, w, lens, tables = cache
    g = torch.Generator(device=DEV).manual_seed(21)
    random = torch.rand(w.shape, device=DEV, generator=g)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_(torch.randint(0, 4, w.shape, device=DEV, generator=g))
    elif kind == "zeros":
        w.mul_(random < 0.1)
    elif kind == "odd":
        w[random < 0.3], w[random < 0.2], w[random < 0.1] = math.inf, math.nan, -math.inf
        w[random > 0.95] = -math.nan
    elif kind == "close":
        w.copy_((torch.full(w.shape, 1.0, device=DEV).view(torch.int32) + (random * 5).int()).view(torch.float32))
    elif kind == "halves":  # all within a part of the range, more than are collected
        w.copy_(1 + random * 2**-12)
        w.view(-1)[::997] = 1e30
    elif kind in ("rising", "falling"):
        for row, n in zip(tables.tolist(), context):
            for i in range(-(-n // 32)):
                at = torch.arange(32, device=DEV) + 32 * i + 1.0
                w[row[i]] = at if kind == "rising" else 1 / at
    if kind == "any":
        tables[6, 300], tables[7, 624] = -1, k.shape[0]
    check(cache, context, [20000, 4000, 8191, 20, 0, 1, 16000, 300], 250)


@pytest.mark.parametrize("context,keep,recent", [([50000], 49999, 0), ([50000], 0, 0), ([50000], 1, 0), ([50000], 700, 700),
                                                 ([50000], 40000, 39990), ([32769], 32768, 1), ([40960, 40961], 8192, 0)])
def test_long_contexts_in_parts_at_their_ends(context, keep, recent):
    check(make_cache(context, page=64, kv_heads=1, seed=22), context, keep, recent)


def test_a_bound_beyond_the_parts():
    """The longest contexts that are allowed for, whatever the requests hold."""
    k, v, weights, lens, tables = make_cache([9000, 100], page=1024, kv_heads=2, seed=23, width=600)
    check((k, v, weights, lens, tables), [9000, 100], 500, 20)
    k, v, weights, lens, tables = make_cache([40000, 9000], page=1024, kv_heads=65, seed=24)  # many heads
    check((k, v, weights, lens, tables), [40000, 9000], 5000, 20)


@pytest.mark.parametrize("dim", [64, 128])
def test_more_rows_than_the_caches_hold(dim):
    """By the bound on what may move; the requests are of every kind."""
    context = [9000, 8001, 8000, 300, 0]
    check(make_cache(context, page=1024, kv_heads=8, dim=dim, seed=25, width=20), context, 8000, 700)


def test_a_long_recent_part_moves_over_itself():
    for shift in (1, 3, 129, 1000):
        context = [4000 + shift]
        check(make_cache(context, dim=128, seed=5), context, 4000, 4000)


def test_requests_that_are_left_as_they_are():
    """Too long, of negative length, or of pages that the cache does not have; their neighbours are cut."""
    page, context = 8, [100, 100, -5, 100, 100, 100]
    k, v, weights, lens, tables = make_cache(context, page=page, seed=6)
    tables[1, 3], tables[3, 12], tables[4, 0] = -1, k.shape[0], 2**31 - 1
    lens[5] = context[5] = 97
    check((k, v, weights, lens, tables), context, 40, 5)
    context = [100, 64, 65]
    check(make_cache(context, page=page, seed=7), context, 20, 5, max_context=64)
    # an entry behind the request's last page says nothing
    k, v, weights, lens, tables = make_cache([30], page=page, seed=8, width=6)
    tables[0, 4:] = i32([-7, 99999])
    check((k, v, weights, lens, tables), [30], 10, 3)


def test_cut_again_after_new_tokens():
    """Rounds of new tokens and cuts: each leaves what the loop leaves."""
    page, keep, recent = 16, 120, 30
    k, v, weights, lens, tables = make_cache([200, 90, 300], page=page, seed=9, kv_heads=3)
    g = torch.Generator(device=DEV).manual_seed(10)
    context = [200, 90, 300]
    for _ in range(4):
        check((k, v, weights, lens, tables), context, keep, recent)
        for b in range(3):
            kept = min(context[b], keep)
            room = [200, 90, 300][b]
            context[b] = min(room, kept + 37)
            at = torch.arange(kept, context[b], device=DEV)
            of, slot = tables[b].long()[at // page], at % page
            for x in (k, v):
                x[of, slot] = torch.randn(len(at), 3, 64, device=DEV, generator=g).to(torch.bfloat16)
            weights[of, :, slot] = torch.rand(len(at), 3, device=DEV, generator=g)
        lens = i32(context)


def test_many_requests():
    g = torch.Generator().manual_seed(11)
    context = torch.randint(0, 200, (700,), generator=g).tolist()
    check(make_cache(context, page=8, kv_heads=1, seed=12), context, 60, 9)


def test_past_32_bit_offsets():
    """Pages whose offsets pass 2^31 elements and 2^32 bytes."""
    pages, page, kv_heads, dim, n, keep, recent = 140000, 16, 8, 128, 100, 40, 10
    both = torch.empty(pages, 2, page, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
    weights = torch.zeros(pages, kv_heads, page, device=DEV)
    entries = [139993 + i if i % 2 else i for i in range(7)]
    tables, g = i32([entries]), torch.Generator(device=DEV).manual_seed(13)
    used = torch.tensor(entries, device=DEV)
    both[used] = torch.randn(7, 2, page, kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    weights[used] = torch.rand(7, kv_heads, page, device=DEV, generator=g)
    small = both[used].clone()
    want = expected(small[:, 0], small[:, 1], weights[used], [n], i32([list(range(7))]), keep, recent)
    got = smx.paged_evict(both[:, 0], both[:, 1], weights, i32([n]), tables, keep, recent=recent)
    assert got.tolist() == [keep]
    assert same(both[used][:, 0], want[0]) and same(both[used][:, 1], want[1]) and same(weights[used], want[2])


@pytest.mark.parametrize("context", [[500, 77, 900], [40000, 33]])
def test_in_a_graph_and_on_two_streams(context):
    first = make_cache(context, seed=14)
    second = make_cache(context, seed=15)
    masters = [[x.clone() for x in c[:3]] for c in (first, second)]
    wants = [expected(*c[:3], context, c[4], 200, 20) for c in (first, second)]
    graphs, lens = [], []
    for c in (first, second):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lens.append(smx.paged_evict(*c, 200, recent=20))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for c, m in zip((first, second), masters):
            for x, y in zip(c, m):
                x.copy_(y)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c, want, n in zip((first, second), wants, lens):
            assert n.tolist() == want[3]
            assert same(c[0], want[0]) and same(c[1], want[1]) and same(c[2], want[2])
        x = torch.randn(1000, 1000, device=DEV)  # the program's own work between replays
        (x @ x).sum().item()


def test_refusals():
    k, v, weights, lens, tables = make_cache([40, 9], page=8)
    for change, message in (
            (dict(k=k.float()), "k_cache"), (dict(v=v[:-1]), "same shape"), (dict(v=k), "keys and values"), (dict(weights=weights[:-1]), "key_weights"),
            (dict(weights=weights.double()), "key_weights"), (dict(weights=weights.transpose(0, 1).contiguous().transpose(0, 1)), "key_weights"),
            (dict(lens=lens.long()), "context_lens"), (dict(lens=lens[:1]), "block_tables"), (dict(tables=tables.long()), "block_tables"),
            (dict(keep=-1), "keep"), (dict(keep=i32([1])), "keep"), (dict(keep=torch.tensor([1, 2], device=DEV)), "keep"),
            (dict(recent=-1), "recent"), (dict(max_context=41), "max_context"), (dict(max_context=-1), "max_context"),
            (dict(lens=lens.cpu()), "HIP device"), (dict(k=k.clone().requires_grad_()), "gradients")):
        args = {"k": k, "v": v, "weights": weights, "lens": lens, "tables": tables, "keep": 8, **change}
        with pytest.raises(ValueError, match=message):
            smx.paged_evict(args.pop("k"), args.pop("v"), args.pop("weights"), args.pop("lens"), args.pop("tables"), args.pop("keep"), **args)
    with pytest.raises(TypeError):
        smx.paged_evict(k, v, weights, lens, tables, 3.5)
    versions = [x._version for x in (k, v, weights)]
    smx.paged_evict(k, v, weights, lens, tables, 8)
    assert all(x._version > y for x, y in zip((k, v, weights), versions))
