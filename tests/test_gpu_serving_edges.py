"""Calls of the serving operators at the edge of what they take, on the GPU: what is refused, and
results where lengths, values and layouts are odd."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import strassen_tpu_amd as smx
from test_gpu_int4 import check, weight
from test_gpu_paged import attend64, check_attention, i32, make_step
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def bf16(*shape, g=None):
    return torch.randn(*shape, device=DEV, generator=g).to(torch.bfloat16)


def test_attention_refuses_results_that_overlap():
    plan, k, v, *_, g = make_step([9], [4], page=8, kv_heads=2, dim=128)
    rows = bf16(5, 8, 128, g=g)
    flat = bf16(5 * 8 * 128, g=g)
    for q, out, message in (
            (rows[:4], rows[1:], "queries"), (rows[1:], rows[:4], "queries"),
            (rows[:4, :4], rows[:4, 2:6], "queries"),
            (rows[:4], flat.as_strided((4, 8, 128), (512, 128, 1)), "on each other"),
            (rows[:4, :2], k.flatten(0, 1)[:4], "cache"), (rows[:4, :2], v.flatten(0, 1)[8:12], "cache")):
        with pytest.raises(ValueError, match=message):
            smx.paged_attention(q, k, v, plan, out=out)


@pytest.mark.parametrize("max_new", [None, 1])
def test_attention_into_columns_beside_the_queries(max_new):
    """Queries and result interleaved in one tensor's memory, row by row, share none of it."""
    context, new = [3000, 12, 90], [1, 1, 1]
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=2, dim=128, pad=2)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    both = bf16(plan.tokens, 16, 128, g=g)
    want, size = attend64(both[:, :8], keys, values, context, new, None)
    kept = both.clone()
    smx.paged_attention(both[:, :8], k, v, plan, out=both[:, 8:])
    check_attention(both[:3, 8:], want[:3], size[:3])
    assert torch.equal(both[:, :8], kept[:, :8]) and torch.equal(both[3:], kept[3:])


def test_write_refuses_overlaps():
    plan, k, v, *_, g = make_step([9], [4], page=8, kv_heads=2, dim=128)
    heads, rows = bf16(4, 2, 128, g=g), k.flatten(0, 1)
    for args, message in (((heads, heads, k, k), "keys and values"), ((rows[:4], heads, k, v), "heads must share"),
                          ((heads, v.flatten(0, 1)[3:7], k, v), "heads must share")):
        with pytest.raises(ValueError, match=message):
            smx.paged_write(*args, plan)
    with pytest.raises(ValueError, match="heads must share"):
        smx.paged_write(heads, heads, k, v, plan, q=rows[8:12])
    near = torch.zeros(k.numel(), dtype=torch.bfloat16, device=DEV).as_strided(k.shape, (k.stride(0) - 128, *k.stride()[1:]))
    with pytest.raises(ValueError, match="each other"):
        smx.paged_write(heads, heads, near, torch.zeros_like(k).as_strided(k.shape, near.stride()), plan)
    # one tensor for both, heads outside the page's tokens: no row of one is a row of the other
    both = torch.zeros(k.shape[0], 2, 2, 8, 128, dtype=torch.bfloat16, device=DEV)
    apart = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    smx.paged_write(heads, heads, *apart, plan)
    at = plan.slots // 8, plan.slots % 8
    assert all(torch.equal(x[at], heads) for x in apart) and int(both.count_nonzero()) == 2 * int(heads.count_nonzero())


def test_plan_refuses_tables_over_its_lists():
    lens, tables = i32([1, 2]), i32([[0, -1, 9, 9], [1, -1, 9, 9]])
    good = dict(page_size=8, num_pages=4, tokens=5, free_pages=i32([2, 3]))
    for args, change in (((lens, lens, tables), {"free_pages": tables[1]}), ((tables[0, :2], lens, tables), {}),
                         ((lens, tables.view(-1)[3:5], tables), {})):
        with pytest.raises(ValueError, match="block_tables"):
            smx.paged_plan(*args, **{**good, **change})
    # a list between the rows of narrower tables, and tables that are only read
    assert smx.paged_plan(lens, lens, tables[:, :2], **{**good, "free_pages": tables[0, 2:]}).status.tolist() == [0, 0]
    assert smx.paged_plan(lens, lens, tables, **{**good, "free_pages": None}).status.tolist() == [0, 0]


@pytest.mark.parametrize("heads,kv_heads", [(64, 1), (128, 1), (8, 2)])
def test_attention_of_a_plan_without_new_tokens(heads, kv_heads):
    """max_new=0: every request sits the step out, whatever the number of query heads to a tile of rows."""
    context = [30, 0, 7]
    plan, k, v, *_, g = make_step(context, [0, 0, 0], page=8, kv_heads=kv_heads, dim=128, pad=5)
    plan = smx.paged_plan(i32(context), i32([0, 0, 0]), plan.block_tables, page_size=8, num_pages=plan.num_pages,
                          tokens=5, max_new=0)
    assert plan.status.tolist() == [smx.PAGED_OK] * 3
    q = bf16(plan.tokens, heads, 128, g=g)
    assert not smx.paged_attention(q, k, v, plan).any()
    out = torch.full_like(q, 7.0)
    assert (smx.paged_attention(q, k, v, plan, out=out) == 7).all()


def test_int4_operands_that_do_not_hold_what_they_say():
    """Fields and tensors changed by hand: sizes that the kernels would read past are refused before a launch."""
    codes, scales, zero, w, spread, g = weight(256, 70, 64, True)
    good = smx.int4_weight_layout(codes, scales, zero, group=64)
    x = bf16(3, 256, g=g)
    for change, message in (
            ({"codes": good.codes[:-1]}, "w.codes"), ({"codes": good.codes.float()}, "w.codes"), ({"codes": good.codes.cpu()}, "on"),
            ({"codes": good.codes.transpose(0, 1)}, "w.codes"), ({"scales": good.scales[:, :1]}, "w.scales"),
            ({"scales": good.scales.short()}, "w.scales"), ({"scales": good.scales.cpu()}, "w.scales"), ({"n": 97}, "w.codes"),
            ({"n": 0}, "w.n"), ({"n": 1 << 40}, "w.n"), ({"k": 288}, "w.codes"), ({"k": -32}, "w.k"), ({"group": 32}, "w.scales"),
            ({"group": 96}, "w.group"), ({"group": 0}, "w.group")):
        fields = {f: getattr(good, f) for f in ("codes", "scales", "k", "n", "group", "swiglu", "zeros")}
        made = smx.Int4Operand(**{**fields, **change})
        with pytest.raises(ValueError, match=message):
            smx.int4_matmul(x, made)
    made = smx.Int4Operand(good.codes.clone(), good.scales.flatten(), 256, 70, 64, False, True)  # by hand, but right
    check(smx.int4_matmul(x, made), x, w, spread)


def write_inputs(g):
    """A plan, its cache and every tensor that paged_write takes."""
    plan, k_cache, v_cache, *_ = make_step([9], [4], page=8, kv_heads=2, dim=128)
    angle = torch.rand(plan.max_context, 64, device=DEV, generator=g)
    return plan, dict(k=bf16(4, 2, 128, g=g), v=bf16(4, 2, 128, g=g), k_cache=k_cache, v_cache=v_cache, q=bf16(4, 8, 128, g=g),
                      rope_cos=angle.cos(), rope_sin=angle.sin(), q_scale=bf16(128, g=g), k_scale=bf16(128, g=g))


def test_write_refuses_gradients_of_all_its_tensors():
    """Norm weights, a model's parameters, among them; without gradients to record they are taken."""
    plan, good = write_inputs(torch.Generator(device=DEV).manual_seed(1))
    want = smx.paged_write(plan=plan, **good)
    for name in good:
        args = {**good, name: good[name].clone().requires_grad_()}
        with pytest.raises(ValueError, match="gradients"):
            smx.paged_write(plan=plan, **args)
        with torch.no_grad():
            assert torch.equal(smx.paged_write(plan=plan, **args), want)


def test_tangents_are_refused():
    """Forward-mode gradients, which torch.no_grad() leaves on."""
    plan, good = write_inputs(torch.Generator(device=DEV).manual_seed(2))
    codes, scales, zero, *_, g = weight(128, 40, 128, True)
    w = smx.int4_weight_layout(codes, scales, zero, group=128)
    x, bias, residual = bf16(4, 128, g=g), bf16(40, g=g), bf16(4, 40, g=g)
    q, k, v = (good[n] for n in ("q", "k_cache", "v_cache"))
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        calls = [lambda n=n: smx.paged_write(plan=plan, **{**good, n: dual(good[n])}) for n in good]
        calls += [lambda: smx.paged_attention(dual(q), k, v, plan), lambda: smx.paged_attention(q, dual(k), v, plan),
                  lambda: smx.paged_attention(q, k, dual(v), plan), lambda: smx.paged_attention(q, k, v, plan, out=dual(q)),
                  lambda: smx.int4_matmul(dual(x), w),
                  lambda: smx.int4_matmul(x, w, epilogue="bias_add", bias=dual(bias)),
                  lambda: smx.int4_matmul(x, w, epilogue="residual_add", residual=dual(residual))]
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        smx.paged_attention(smx.paged_write(plan=plan, **good), k, v, plan)
        smx.int4_matmul(forward_ad.unpack_dual(dual(x)).primal, w)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,new,max_new,window", [
    ([0, 20, 9000], [1, 1, 1], 1, None), ([5, 0, 3000], [3, 4, 1], 4, 1), ([0, 40, 6000], [150, 70, 9], None, None),
    ([90, 700], [150, 70], None, 33)])
def test_attention_of_infinite_scores(dim, context, new, max_new, window):
    """Infinities among the keys. A score of -inf weighs nothing beside others; a row that sees no other score is NaN
    (not the zero of a row that sees no key), and so is one that sees a score of +inf."""
    page, kv_heads, heads = 8, 3, 6
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, pad=2)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = bf16(plan.tokens, heads, dim, g=g)
    q[:, :, 5] = q[:, :, 5].abs() + 1  # the sign of the infinity is the score's
    for b, (c, n) in enumerate(zip(context, new)):
        at = torch.arange(c + n, device=DEV)
        rows = plan.block_tables[b].long()[at // page], at % page
        odd = torch.zeros(c + n, kv_heads, device=DEV)
        odd[::3, 0] = -math.inf  # every third, the first among them
        odd[:c + (n + 1) // 2, 1] = -math.inf  # all that the first half of the rows see
        odd[c + n // 2, 2] = math.inf
        column = torch.where(odd != 0, odd, k[(*rows, slice(None), 5)].float())
        k[(*rows, slice(None), 5)] = column.to(torch.bfloat16)
        keys[b][:, :, 5] = column.double()
    want, size, row = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV), 0
    for b, (c, n) in enumerate(zip(context, new)):
        key, own = torch.arange(c + n, device=DEV), torch.arange(c, c + n, device=DEV)[:, None]
        hidden = (key > own) | (key <= own - (window or 1 << 30))
        for h in range(heads):
            # elementwise, not by a library product, whose sums of infinities are its own affair
            s = (q[row:row + n, h, None].double() * keys[b][None, :, h // 2]).sum(-1) * dim ** -0.5
            w = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
            want[row:row + n, h], size[row:row + n, h] = w @ values[b][:, h // 2], w @ values[b][:, h // 2].abs()
        row += n
    got = smx.paged_attention(q, k, v, plan, window=window)
    assert torch.equal(got.isnan(), want.isnan())
    assert want.isnan().any() and not want[row:].any()
    here = ~want.isnan()
    check_attention(got[here], want[here], size[here])


@pytest.mark.parametrize("max_new", [None, 2])
def test_attention_of_a_row_that_sees_infinite_scores_and_missing_pages(max_new):
    """Rows whose pages are all missing are zero, those that see one key of score -inf among missing pages NaN."""
    context, new, page = [40, 16], [2, 2], 8
    plan, k, v, *_, g = make_step(context, new, page=page, kv_heads=1, dim=128)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = bf16(4, 2, 128, g=g).abs() + 1
    k.copy_(torch.where(k.isnan(), k, torch.full_like(k, -math.inf)))
    plan.block_tables[0], plan.block_tables[1, 1:] = -1, plan.num_pages
    for window in (None, 12):
        got = smx.paged_attention(q, k, v, plan, window=window)
        assert not got[:2].any()
        # positions 16 and 17 of the second request see keys 5 .. and 6 .. of the page that is there
        assert got[2:].isnan().all()
    assert not smx.paged_attention(q, k, v, plan, window=8).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,new,max_new,window", [
    ([3, 41, 2000], [1, 1, 1], 1, None), ([30, 5, 200], [4, 3, 4], 4, 8), ([0, 100], [150, 70], None, None),
    ([90, 700], [150, 70], None, 33)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_attention_of_infinities_whose_weight_is_nothing(dim, context, new, max_new, window, value):
    """A key 300 below the others, whose weight FP32 does not hold: an infinity or NaN of its value reaches the rows
    that see it all the same, in steps that mask keys and in others, and no other row."""
    page, heads = 8, 4
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=1, dim=dim)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = bf16(plan.tokens, heads, dim, g=g)
    q[:, :, 5] = 2.0
    reached, row = torch.zeros(plan.tokens, dtype=torch.bool, device=DEV), 0
    for b, (c, n) in enumerate(zip(context, new)):
        own = torch.arange(c, c + n, device=DEV)
        for at in {max(0, c - 2), max(0, c + n // 2 - 1)}:
            page_at = plan.block_tables[b, at // page]
            k[page_at, at % page, 0, 5], v[page_at, at % page, 0, 17] = -2400.0 * (dim / 64) ** 0.5, value
            reached[row:row + n] |= (at <= own) & (at > own - (window or 1 << 30))
        row += n
    got = smx.paged_attention(q, k, v, plan, window=window)[:, :, 17]
    assert (~got.isfinite()).eq(reached[:, None]).all() and reached.any()


@pytest.mark.parametrize("requests,page,most,tokens", [(5, 8, 70, 400), (70, 8, 40, 4000), (1500, 16, 70, 60000), (3, 8, 9000, 30000)])
def test_plan_without_a_free_list_looks_at_every_page_of_the_new_tokens(requests, page, most, tokens):
    """Missing entries among the pages that the new tokens go to, a few or thousands of a request, keep it out; entries
    before and behind them do not matter."""
    g = torch.Generator().manual_seed(requests)
    context = torch.randint(0, 60, (requests,), generator=g)
    new = torch.randint(0, most, (requests,), generator=g)
    context[0], new[0] = 2 * page, page  # whole pages
    width = int(((context + new + page - 1) // page).max()) + 1
    pages = requests * width
    tables = torch.randperm(pages, generator=g).view(requests, width)
    first, last = context // page, (context + new - 1) // page
    at = torch.arange(width)[None]
    tables[(at < first[:, None]) | (at > last[:, None])] = -1  # what no new token goes to
    bad = torch.rand(requests, generator=g) < 0.5
    bad[0] = False
    where = first + (torch.rand(requests, generator=g) * (last - first + 1)).long()
    where[1], where[2] = first[1], last[2]
    odd = torch.tensor([-1, pages, 2**31 - 1, -2**31])[torch.arange(requests) % 4]
    spoilt = bad & (new > 0)
    tables[spoilt, where[spoilt]] = odd[spoilt]
    plan = smx.paged_plan(i32(context.tolist()), i32(new.tolist()), i32(tables.tolist()), page_size=page, num_pages=pages,
                          tokens=tokens)
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0)))
    assert int(starts[-1]) <= tokens and spoilt.any()
    assert plan.status.tolist() == torch.where(spoilt, smx.PAGED_BAD_PAGE, smx.PAGED_OK).tolist()
    assert plan.rows.tolist() == torch.where(spoilt, 0, new).tolist() and plan.starts.tolist() == starts.tolist()
    slots = torch.full((tokens,), -1)
    for b in range(requests):
        if not spoilt[b]:
            key = torch.arange(int(context[b]), int(context[b] + new[b]))
            slots[starts[b]:starts[b + 1]] = tables[b][key // page] * page + key % page
    assert plan.slots.tolist() == slots.tolist()  # no row of an admitted request without a place
    assert torch.equal(plan.positions >= 0, plan.slots >= 0)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m,zeros", [(1, True), (20, True), (61, False)])
def test_int4_of_the_largest_values(group, m, zeros):
    """|x| up to 2^115 times scales that bring the sums back: 128 terms of 31 |x| stay below 2^127."""
    codes, scales, zero, w, spread, g = weight(512, 70, group, zeros)
    scales = (scales.float() * 2.0 ** -118).to(torch.bfloat16)  # some of them subnormal, with fewer bits
    spread = scales.double().repeat_interleave(group, 0)
    w = (codes.double() - (8 if zero is None else zero.double().repeat_interleave(group, 0))) * spread
    laid = smx.int4_weight_layout(codes, scales, zero, group=group)
    x = bf16(m, 512, g=g).sign() * 2.0 ** 115  # of one size: the sums are as large as they get
    x[0] = x[0].abs()  # without cancellation
    check(smx.int4_matmul(x, laid), x, w, spread.abs())


def counted_cache(context, new, *, page, kv_heads, dim, seed, max_new=None):
    """A plan, and a cache whose values are whole numbers in a few units: with queries of zero every key weighs 1, so
    that a row's sums are exact in FP32 and its result is their mean, rounded once. Also the requests' values
    summed up to each position [context + new, kv_heads, dim]."""
    plan, k, v, keys, values, g = make_step(context, new, page=page, kv_heads=kv_heads, dim=dim, seed=seed)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=page, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    sums = []
    for b, (c, n) in enumerate(zip(context, new)):
        at = torch.arange(c + n, device=DEV)
        whole = torch.randint(-8, 9, (c + n, kv_heads, dim), device=DEV, generator=g).double()
        v[plan.block_tables[b].long()[at // page], at % page] = whole.to(torch.bfloat16)
        sums.append(whole.cumsum(0))
    return plan, k, v, sums


def check_means(got, sums, context, new, window, steps):
    """Every row's mean over the keys that it sees, to one rounding (and the reciprocal's): a step of keys left out,
    counted twice or taken from elsewhere moves a row's 64 or more columns by several times that."""
    row = 0
    for (c, n), total in zip(zip(context, new), sums):
        own = torch.arange(c, c + n, device=DEV)
        seen = torch.clamp(own + 1, max=window or 1 << 30)
        before = torch.where((own >= seen)[:, None, None], total[(own - seen).clamp(min=0)], 0.0)
        want = (total[own] - before) / seen[:, None, None]
        mine = got[row:row + n].double().unflatten(1, (total.shape[1], -1))
        bound = (2.0 ** -8 + 2.0 ** -22) * want.abs()[:, :, None]
        assert ((mine - want[:, :, None]).abs() <= bound).all()
        # what the bound can tell, for the last row: any one step of its keys left out
        first, last = int(own[-1] - seen[-1]) // steps + 1, int(own[-1]) // steps
        ends = total[torch.arange(first + 1, max(first + 1, last), device=DEV) * steps - 1]  # (none of a short one)
        lost = want[-1] - (want[-1] * seen[-1] - ends.diff(dim=0)) / (seen[-1] - steps)
        assert (lost.abs() > 2 * bound[-1, :, 0]).flatten(1).any(1).all()
        row += n


@pytest.mark.parametrize("context,new,kv_heads,group,dim,max_new,window", [
    ([131000], [1], 1, 8, 128, 1, None), ([131071, 5, 70001, 129], [1, 1, 1, 1], 2, 4, 64, 1, None),
    ([131000, 3000], [4, 3], 1, 8, 128, 4, None), ([131000, 65536], [1, 1], 2, 8, 128, 1, 70000),
    ([131000], [40], 1, 4, 128, None, None), ([131071, 9, 40000], [1, 1, 300], 2, 8, 64, None, None),
    ([131000, 65530], [200, 33], 1, 4, 64, None, 70000), ([1_000_000], [1], 1, 2, 128, 1, None)])
def test_attention_counts_every_key_of_long_contexts(context, new, kv_heads, group, dim, max_new, window):
    plan, k, v, sums = counted_cache(context, new, page=64, kv_heads=kv_heads, dim=dim, seed=11, max_new=max_new)
    q = torch.zeros(plan.tokens, kv_heads * group, dim, dtype=torch.bfloat16, device=DEV)
    check_means(smx.paged_attention(q, k, v, plan, window=window), sums, context, new, window, 32 if max_new else 64)


@pytest.mark.parametrize("window", [None, 20000])
def test_attention_counts_every_key_of_a_long_prompt(window):
    """All of 100,000 rows, whose tiles' counts of steps pass 16 bits."""
    plan, k, v, sums = counted_cache([0], [100_000], page=64, kv_heads=1, dim=64, seed=12)
    q = torch.zeros(plan.tokens, 2, 64, dtype=torch.bfloat16, device=DEV)
    check_means(smx.paged_attention(q, k, v, plan, window=window), sums, [0], [100_000], window, 64)


@pytest.mark.parametrize("context,new,max_new,dim", [([131000, 20], [1, 1], 1, 128), ([131072], [1], 1, 64),
                                                    ([131000, 20], [30, 1], None, 128)])
def test_attention_of_131000_keys(context, new, max_new, dim):
    """Weights and result are rounded to bf16, each by half a step at most evenly spread, 2^-8 / 3^0.5 in the mean:
    2^-8 (2 / 3)^0.5 = 3.2e-3 of a row's norm together, over 64 or more columns seldom more than a third above it. A
    step of 32 keys less would be (32 / 131000)^0.5 = 1.6e-2."""
    plan, k, v, keys, values, g = make_step(context, new, page=16, kv_heads=2, dim=dim, seed=13)
    plan = smx.paged_plan(i32(context), i32(new), plan.block_tables, page_size=16, num_pages=plan.num_pages,
                          tokens=plan.tokens, max_new=max_new)
    q = bf16(plan.tokens, 8, dim, g=g)
    want, size = attend64(q, keys, values, context, new, None)
    got = smx.paged_attention(q, k, v, plan)
    check_attention(got, want, size)
    assert ((got.double() - want).norm(dim=-1) <= 5e-3 * want.norm(dim=-1)).all()


def test_backward_passes_find_out_what_was_written():
    """Values kept for a backward pass that a call overwrites are an error there, not another gradient."""
    plan, good = write_inputs(torch.Generator(device=DEV).manual_seed(3))
    k_cache, v_cache, q = good["k_cache"], good["v_cache"], good["q"]
    out, tables = torch.zeros_like(q), i32([[0, 1, -1]])
    lens = i32([9])
    for kept, call in ((k_cache, lambda: smx.paged_write(plan=plan, **good)), (v_cache, lambda: smx.paged_write(plan=plan, **good)),
                       (out, lambda: smx.paged_attention(q, k_cache, v_cache, plan, out=out)),
                       (tables, lambda: smx.paged_plan(lens, lens, tables, page_size=8, num_pages=4, tokens=9, free_pages=i32([3])))):
        factor = torch.ones((), device=DEV, requires_grad=True)
        loss = (factor * kept).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    assert tables.tolist() == [[0, 1, 3]]
    before = tables._version, k_cache._version, q._version
    smx.paged_plan(lens, lens, tables, page_size=8, num_pages=4, tokens=9)  # read only
    smx.paged_attention(q, k_cache, v_cache, plan)
    assert before == (tables._version, k_cache._version, q._version)
    with torch.inference_mode():
        cache = [torch.zeros_like(k_cache) for _ in range(2)]
    with torch.no_grad():  # tensors of inference mode, which count no versions
        smx.paged_write(good["k"], good["v"], *cache, plan)
    assert torch.equal(cache[0][plan.slots // 8, plan.slots % 8], good["k"])
