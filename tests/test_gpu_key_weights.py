"""The attention weight that cached keys receive, and the logarithms of the attention's sums, on the GPU against their
definitions in 64 bits."""

import math

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_paged import attend64, check_attention, i32, make_step
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def weights64(q, keys, context, new, window, scale, before, unseen=()):
    """Each row's logarithm of its sum, and by request the keys' weights [kv_heads, context + new] after the step."""
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    after, row = [], 0
    for b, (c, n) in enumerate(zip(context, new)):
        found = before[b].double().clone()
        found[:, c:] = 0 if n else found[:, c:]
        key, own = torch.arange(c + n, device=DEV), torch.arange(c, c + n, device=DEV)[:, None]
        hidden = key > own
        if window:
            hidden = hidden | (key <= own - window)
        for bb, j in unseen:
            if bb == b:
                hidden = hidden | (key == j)
        group = q.shape[1] // found.shape[0]
        for h in range(q.shape[1] if n else 0):
            score = (scale * (q[row:row + n, h].double() @ keys[b][:, h // group].t())).masked_fill(hidden, -math.inf)
            lse[row:row + n, h] = torch.logsumexp(score, -1)
            found[h // group] += torch.softmax(score, -1).nan_to_num(0.0).sum(0)
        after.append(found)
        row += n
    return lse, after


def received(weights, tables, b, length):
    at = torch.arange(length, device=DEV)
    page = weights.shape[2]
    return weights[tables[b].long()[at // page], :, at % page].t()  # [kv_heads, length]


def check(plan, k, v, keys, g, context, new, heads, *, window=None, scale=None, fill=None, size=1.0):
    dim, kv_heads, page = k.shape[3], k.shape[2], k.shape[1]
    q = (size * torch.randn(plan.tokens, heads, dim, device=DEV, generator=g)).to(torch.bfloat16)
    weights = torch.rand(k.shape[0], kv_heads, page, device=DEV, generator=g) if fill is None else fill
    before = [received(weights, plan.block_tables, b, c + n) for b, (c, n) in enumerate(zip(context, new))]
    lse = torch.full((plan.tokens, heads), 7.0, device=DEV)
    kept = weights.clone()
    out = smx.paged_attention(q, k, v, plan, window=window, scale=scale, lse=lse)
    assert torch.equal(out, smx.paged_attention(q, k, v, plan, window=window, scale=scale))
    smx.paged_key_weights(q, k, weights, plan, lse, window=window, scale=scale)
    want_lse, want = weights64(q, keys, context, new, window, dim ** -0.5 if scale is None else scale, before)
    used = sum(new)
    # A score is a sum of up to 128 products in FP32, off by 128 2^-24 of the sum of their sizes at most; these are below
    # 16 (here |q| |k| scale), 1.2e-4. The sum of exponentials and its logarithm add a part of that.
    assert ((lse[:used].double() - want_lse[:used]).abs() <= 2e-4).all()
    assert (lse[used:] == 7).all()
    untouched = torch.ones_like(weights, dtype=torch.bool)
    for b, (c, n) in enumerate(zip(context, new)):
        got = received(weights, plan.block_tables, b, c + n).double()
        # the same off in score and lse, and a rounding for each addition's running sum
        assert ((got - want[b]).abs() <= (4e-4 + 2**-24 * (2 * n * heads // kv_heads + 2)) * want[b] + 1e-30).all(), b
        if n:
            at = torch.arange(c + n, device=DEV)
            untouched[plan.block_tables[b].long()[at // page], :, at % page] = False
    assert torch.equal(weights[untouched], kept[untouched])
    return q, weights, lse


CASES = [
    # context, new, page, heads, kv_heads, dim, window, max_new, layout
    ([0], [1], 16, 1, 1, 64, None, 1, "pages"), ([0, 0], [1, 3], 8, 8, 2, 128, None, None, "pages"),
    ([1000], [1], 16, 64, 8, 128, None, 1, "pages"), ([31, 32, 33, 255, 256, 257], [1] * 6, 16, 16, 2, 128, None, 1, "heads"),
    ([300, 0, 77], [1, 2, 0], 8, 32, 2, 64, None, 2, "one"), ([700, 3, 40], [4, 3, 4], 32, 8, 1, 128, 50, 4, "pages"),
    ([5000, 100], [1, 1], 64, 8, 8, 128, 1, 1, "pages"), ([600, 90], [1, 1], 16, 8, 2, 64, 256, 1, "pages"),
    # many rows
    ([0], [300], 16, 8, 2, 128, None, None, "pages"), ([0, 513, 100], [40, 257, 1], 16, 6, 2, 64, None, None, "heads"),
    ([255, 256, 257], [33, 1, 70], 8, 10, 2, 128, None, None, "one"), ([2000], [500], 128, 16, 2, 128, 300, None, "pages"),
    ([100, 1000], [700, 20], 16, 4, 1, 64, 64, None, "pages"), ([900, 0], [129, 600], 16, 128, 1, 128, None, None, "pages"),
    ([400], [9], 16, 100, 1, 64, None, None, "pages"), ([3000], [64], 16, 8, 8, 128, 1, None, "pages"),
    ([0, 0], [1, 1], 8, 40, 8, 128, None, None, "pages"), ([70], [5], 16, 33, 1, 64, 2**31 - 1, 5, "pages"),
]


@pytest.mark.parametrize("context,new,page,heads,kv_heads,dim,window,max_new,layout", CASES)
def test_key_weights(context, new, page, heads, kv_heads, dim, window, max_new, layout):
    plan, k, v, keys, _, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, pad=3, layout=layout)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    check(plan, k, v, keys, g, context, new, heads, window=window)
    check(plan, k, v, keys, g, context, new, heads, window=window, scale=0.3, size=0.3)


@pytest.mark.parametrize("new_high,max_new", [(1, 1), (3, 4), (3, None)])
@pytest.mark.parametrize("window", [None, 40])
def test_many_requests(new_high, max_new, window):
    """More requests than a workgroup looks at in one round, some of them idle."""
    generator = torch.Generator().manual_seed(7)
    context = torch.randint(0, 150, (700,), generator=generator).tolist()
    new = torch.randint(0, new_high + 1, (700,), generator=generator).tolist()
    plan, k, v, keys, _, g = make_step(context, new, page=16, kv_heads=1, dim=64, pad=1)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    check(plan, k, v, keys, g, context, new, 4, window=window)


@pytest.mark.parametrize("context,new,heads,kv_heads,dim,max_new", [([20000], [1], 16, 2, 128, 1), ([9000, 40], [600, 1], 8, 2, 64, None),
                                                                  ([131000], [2], 8, 1, 128, 2), ([0], [5000], 2, 1, 128, None)])
def test_long_contexts(context, new, heads, kv_heads, dim, max_new):
    plan, k, v, keys, _, g = make_step(context, new, page=64, kv_heads=kv_heads, dim=dim)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=64, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    check(plan, k, v, keys, g, context, new, heads)


@pytest.mark.parametrize("max_new", [None, 2])
def test_the_same_bits_again(max_new):
    """Items that several workgroups share are added up in one order."""
    context, new = [4000 + b for b in range(12)], [2] * 12
    plan, k, v, *_, g = make_step(context, new, page=16, kv_heads=2, dim=128)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = torch.randn(plan.tokens, 16, 128, device=DEV, generator=g).to(torch.bfloat16)
    lse = torch.empty(plan.tokens, 16, device=DEV)
    smx.paged_attention(q, k, v, plan, lse=lse)
    first, other = None, torch.empty(1 << 28, device=DEV)
    for _ in range(8):
        weights = torch.zeros(k.shape[0], 2, 16, device=DEV)
        other.zero_()
        smx.paged_key_weights(q, k, weights, plan, lse)
        first = weights if first is None else first
        assert torch.equal(weights, first)
    # all rows' weights add up to one each: 24 rows of 16 heads
    assert abs(first.double().sum().item() - 24 * 16) <= 24 * 16 * 4e-4


@pytest.mark.parametrize("max_new", [None, 4])
def test_pages_that_are_not_in_the_cache(max_new):
    """Their keys receive nothing and take nothing from others; weights of other slots stay."""
    context, new, page = [40, 2, 120], [2, 3, 1], 8
    plan, k, v, keys, _, g = make_step(context, new, page=page, kv_heads=2, dim=128, pad=2)
    tables = plan.block_tables
    whole = tables.clone()
    plan = smx.paged_plan(i32(context), i32(new), tables, page_size=page, num_pages=plan.num_pages, tokens=plan.tokens, max_new=max_new)
    tables[0, 1], tables[0, 5], tables[1, 0], tables[2, 14] = -1, plan.num_pages, 2**31 - 1, -2**31
    unseen = [(0, j) for j in range(8, 16)] + [(0, j) for j in range(40, 48)] + [(1, j) for j in range(8)]
    unseen += [(2, j) for j in range(112, 120)]
    q = torch.randn(plan.tokens, 8, 128, device=DEV, generator=g).to(torch.bfloat16)
    weights = torch.rand(k.shape[0], 2, page, device=DEV, generator=g)
    kept, lse = weights.clone(), torch.zeros(plan.tokens, 8, device=DEV)
    before = [received(weights, whole, b, c + n) for b, (c, n) in enumerate(zip(context, new))]
    smx.paged_attention(q, k, v, plan, lse=lse)
    smx.paged_key_weights(q, k, weights, plan, lse)
    want_lse, want = weights64(q, keys, context, new, None, 128 ** -0.5, before, unseen)
    seen = want_lse[:6].isfinite()
    assert torch.equal(lse[:6].isfinite(), seen) and ((lse[:6].double() - want_lse[:6])[seen].abs() <= 2e-4).all()
    assert (lse[2:5] == -math.inf).all()  # the second request's rows see nothing
    for b, (c, n) in enumerate(zip(context, new)):
        got, here = received(weights, whole, b, c + n).double(), torch.ones(c + n, dtype=torch.bool, device=DEV)
        here[[j for bb, j in unseen if bb == b and j < c + n]] = False
        assert torch.equal(got[:, ~here], before[b][:, ~here].double())
        assert ((got - want[b])[:, here].abs() <= 5e-4 * want[b][:, here]).all()
    assert torch.equal(weights[~torch.isin(torch.arange(k.shape[0], device=DEV), whole)], kept[~torch.isin(torch.arange(k.shape[0], device=DEV), whole)])


@pytest.mark.parametrize("max_new", [None, 3])
def test_infinities_and_nan_of_the_keys(max_new):
    """A NaN score makes its row's sum NaN, and with it what the keys that the row sees receive; rows that do not see
    it give what they give without it. A score of -inf receives nothing."""
    context, new = [50, 400], [3, 2]
    plan, k, v, keys, _, g = make_step(context, new, page=8, kv_heads=2, dim=64)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=8, num_pages=plan.num_pages, tokens=plan.tokens,
                          max_new=max_new)
    q = torch.rand(plan.tokens, 4, 64, device=DEV, generator=g).to(torch.bfloat16) + 0.1
    lse, weights = torch.zeros(plan.tokens, 4, device=DEV), torch.zeros(k.shape[0], 2, 8, device=DEV)
    k[plan.block_tables[0, 51 // 8], 51 % 8, 0, 7] = math.nan  # the first new token but one: the last two rows see it
    k[plan.block_tables[1, 3], 2, 1, 5] = -math.inf  # every query is positive
    keys[1][26, 1, 5] = -math.inf
    smx.paged_attention(q, k, v, plan, lse=lse)
    smx.paged_key_weights(q, k, weights, plan, lse)
    assert lse[1:3, :2].isnan().all() and lse[:1].isfinite().all() and lse[1:3, 2:].isfinite().all() and lse[3:].isfinite().all()
    got = received(weights, plan.block_tables, 0, 53)
    assert got[0].isnan().all() and got[1].isfinite().all()
    before = [torch.zeros(2, c + n, device=DEV) for c, n in zip(context, new)]
    _, want = weights64(q, [x.nan_to_num(0.0, posinf=0.0, neginf=-math.inf) for x in keys], context, new, None, 64 ** -0.5, before)
    got = received(weights, plan.block_tables, 1, 402).double()
    assert got[1, 26] == 0 and ((got - want[1]).abs() <= 5e-4 * want[1]).all()


def test_lse_of_rows_whose_scores_are_minus_infinity():
    plan, k, v, *_ = make_step([4], [1], page=8, kv_heads=1, dim=64)
    k[plan.block_tables[0].long()] = -math.inf
    lse = torch.zeros(1, 1, device=DEV)
    out = smx.paged_attention(torch.ones(1, 1, 64, dtype=torch.bfloat16, device=DEV), k, v, plan, lse=lse)
    assert lse.item() == -math.inf and out.isnan().all()


def test_requests_that_are_not_admitted():
    context, new = [20, 30, 4], [3, 5, 2]
    plan, k, v, keys, _, g = make_step(context, new, page=8, kv_heads=2, dim=64, pad=1)
    less = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=8, num_pages=plan.num_pages, tokens=plan.tokens, max_new=4)
    q = torch.randn(plan.tokens, 2, 64, device=DEV, generator=g).to(torch.bfloat16)
    results = []
    for p in (plan, less):
        lse, weights = torch.full((p.tokens, 2), 3.0, device=DEV), torch.full((k.shape[0], 2, 8), 5.0, device=DEV)
        smx.paged_attention(q, k, v, p, lse=lse)
        smx.paged_key_weights(q, k, weights, p, lse)
        results.append((lse, weights))
    (lse, weights), (less_lse, less_weights) = results
    assert (less_lse[3:8] == 3).all() and torch.equal(less_lse[:3], lse[:3]) and torch.equal(less_lse[8:10], lse[8:10])
    assert (received(less_weights, plan.block_tables, 1, 35) == 5).all()
    for b, n in ((0, 23), (2, 6)):  # (the kernel for few rows adds in another order)
        assert torch.allclose(received(less_weights, plan.block_tables, b, n), received(weights, plan.block_tables, b, n), rtol=1e-5)


def test_past_32_bit_offsets():
    pages, page, kv_heads, dim = 140000, 16, 8, 128
    both = torch.empty(pages, 2, page, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
    k, v = both[:, 0], both[:, 1]
    g = torch.Generator(device=DEV).manual_seed(3)
    context = [100, 40]
    tables = [[139990 + i if i % 2 else i for i in range(8)], [70000 + i for i in range(3)] + [0] * 5]
    for new, max_new in (([20, 1], None), ([1, 1], 1)):
        plan = smx.paged_plan(i32(context), i32(new), i32(tables), page_size=page, num_pages=pages, tokens=sum(new), max_new=max_new)
        keys = []
        for b, (c, n) in enumerate(zip(context, new)):
            at = torch.arange(c + n, device=DEV)
            x, y = (torch.randn(c + n, kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
            k[i32(tables[b]).long()[at // page], at % page], v[i32(tables[b]).long()[at // page], at % page] = x, y
            keys.append(x.double())
        check(plan, k, v, keys, g, context, new, 16, fill=torch.rand(pages, kv_heads, page, device=DEV, generator=g))


@pytest.mark.parametrize("max_new", [None, 1])
def test_queries_of_odd_strides(max_new):
    """Query heads that are laid out anew, columns of a projection, heads outside the tokens."""
    context, new = [300, 40], [1, 1]
    plan, k, v, *_, g = make_step(context, new, page=16, kv_heads=2, dim=64)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages, tokens=2, max_new=max_new)
    q = torch.randn(2, 8, 64, device=DEV, generator=g).to(torch.bfloat16)
    lse, results = torch.empty(2, 8, device=DEV), []
    wide = torch.zeros(2, 12, 64, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:10] = q
    odd = torch.zeros(2 * 8 * 67 + 1, dtype=torch.bfloat16, device=DEV)[1:].as_strided((2, 8, 64), (8 * 67, 67, 1))
    odd.copy_(q)
    for view in (q, wide[:, 2:10], q.transpose(0, 1).contiguous().transpose(0, 1), odd):
        weights = torch.zeros(k.shape[0], 2, 16, device=DEV)
        smx.paged_attention(view, k, v, plan, lse=lse)
        smx.paged_key_weights(view, k, weights, plan, lse)
        results.append(weights)
    assert all(torch.equal(r, results[0]) for r in results)


@pytest.mark.parametrize("max_new", [None, 1])
@pytest.mark.parametrize("far", ["tokens", "heads"])
def test_queries_far_from_each_other(max_new, far):
    """Strides beyond the kernel's offsets within a step's rows."""
    context, new = [300, 40], [1, 1]
    plan, k, v, *_, g = make_step(context, new, page=16, kv_heads=2, dim=64)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages, tokens=2, max_new=max_new)
    q = torch.randn(2, 8, 64, device=DEV, generator=g).to(torch.bfloat16)
    strides = ((1 << 29) + 8, 64, 1) if far == "tokens" else (64, (1 << 27) + 8, 1)
    view = torch.empty(strides[0] + 7 * strides[1] + 64, dtype=torch.bfloat16, device=DEV).as_strided((2, 8, 64), strides)
    view.copy_(q)
    lse = torch.empty(2, 8, device=DEV)
    smx.paged_attention(q, k, v, plan, lse=lse)
    results = [torch.zeros(k.shape[0], 2, 16, device=DEV) for _ in range(2)]
    for x, weights in zip((q, view), results):
        smx.paged_key_weights(x, k, weights, plan, lse)
    assert torch.equal(*results) and results[0].any()


@pytest.mark.parametrize("max_new", [1, 40])
def test_in_a_graph(max_new):
    """Replays after lengths, tables, queries and keys changed in place, eager work between; two graphs at once keep
    workspaces of their own."""
    g = torch.Generator(device=DEV).manual_seed(5)
    page, pages, kv_heads, dim, heads, tokens = 16, 64, 2, 128, 16, 48
    k, v = (torch.randn(pages, page, kv_heads, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    lens, new = i32([100, 0, 300]), i32([1, 1, 1])
    tables = torch.randperm(60, device=DEV, generator=g).to(torch.int32).view(3, 20)
    q = torch.randn(tokens, heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    captured, eager = torch.zeros(pages, kv_heads, page, device=DEV), torch.zeros(pages, kv_heads, page, device=DEV)

    def step(weights):
        plan = smx.paged_plan(lens, new, tables, page_size=page, num_pages=pages, tokens=tokens, max_new=max_new)
        lse = torch.empty(tokens, heads, device=DEV)
        out = smx.paged_attention(q, k, v, plan, lse=lse)
        smx.paged_key_weights(q, k, weights, plan, lse)
        return out

    step(torch.zeros_like(captured))
    torch.cuda.synchronize()
    graphs = []
    for weights in (captured, torch.zeros_like(captured)):
        graphs.append((torch.cuda.CUDAGraph(), weights))
        with torch.cuda.graph(graphs[-1][0]):
            step(weights)
    side = torch.cuda.Stream()
    for i in range(4):
        want = step(eager).clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager) and torch.equal(graphs[1][1], eager) and want.isfinite().all()
        lens += new
        if max_new > 1:
            new.copy_(i32([[20, 3, 1], [0, 17, 9], [1, 1, 1], [2, 2, 2]][i]))
        tables.copy_(tables.roll(1, 0) if i == 1 else tables)
        q.copy_(torch.randn(tokens, heads, dim, device=DEV, generator=g))


def test_refusals():
    plan, k, v, *_, g = make_step([9], [4], page=8, kv_heads=2, dim=128)
    q, lse = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 8, device=DEV)
    weights = torch.zeros(k.shape[0], 2, 8, device=DEV)
    for change, message in (
            (dict(q=q.float()), "q must"), (dict(q=q[:3]), "q must"), (dict(q=q[:, :7]), "query heads|lse"), (dict(k=k[:-1]), "plan is of"),
            (dict(weights=weights[1:]), "key_weights"), (dict(weights=weights.to(torch.bfloat16)), "key_weights"),
            (dict(lse=lse[:, :4]), "lse"), (dict(lse=lse.double()), "lse"), (dict(lse=lse.t().contiguous().t()), "lse"),
            (dict(scale=0.0), "scale"), (dict(window=0), "window"), (dict(window=2.0), "window"),
            (dict(lse=weights.view(-1)[:32].view(4, 8)), "share no memory"), (dict(q=q.clone().requires_grad_()), "gradients")):
        args = {"q": q, "k": k, "weights": weights, "lse": lse, **change}
        with pytest.raises(ValueError, match=message):
            smx.paged_key_weights(args.pop("q"), args.pop("k"), args.pop("weights"), plan, args.pop("lse"), **args)
    for bad in (lse[:3], lse.double(), lse.cpu(), lse.t().contiguous().t()):
        with pytest.raises(ValueError, match="lse|HIP device"):
            smx.paged_attention(q, k, v, plan, lse=bad)
    with pytest.raises(ValueError, match="lse"):
        out = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device=DEV)
        smx.paged_attention(q, k, v, plan, out=out, lse=out.view(-1).view(torch.float32)[:32].view(4, 8))
    versions = weights._version, lse._version
    smx.paged_attention(q, k, v, plan, lse=lse)
    smx.paged_key_weights(q, k, weights, plan, lse)
    assert weights._version > versions[0] and lse._version > versions[1]
