"""The serving operators one after the other, as a program uses them: drafts verified, keys weighed and caches cut, at positions of the
program's own, against a simulation in 64 bits; and the decoder block's steps with them."""

import dataclasses

import pytest
import torch

import strassen_tpu_amd as smx
import strassen_tpu_amd.qwen3_block as qb
from test_gpu_paged import i32
from test_gpu_parity import DEV, say
from test_gpu_rotary import check, rotate64

pytestmark = pytest.mark.gpu

DIMS = qb.Qwen3Dims(hidden=512, ffn=1024, heads=8, kv_heads=2)
TILE = (256, 256)


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


class Request:
    """A request of the simulation: tokens so far and, for each key/value head, what the cache holds, on the CPU in 64 bits."""

    def __init__(self, kv_heads, dim):
        self.tokens, self.position = [], 0
        self.keys = [torch.zeros(0, dim, dtype=torch.float64) for _ in range(kv_heads)]
        self.values = [torch.zeros(0, dim, dtype=torch.float64) for _ in range(kv_heads)]
        self.weights = [torch.zeros(0, dtype=torch.float64) for _ in range(kv_heads)]


class Program:
    """A model of one attention layer, and its cache: q, k and v are looked up by token, probabilities are the softmax of the
    attended heads times a matrix."""

    def __init__(self, requests, *, heads=8, kv_heads=2, dim=64, page=8, width=12, vocab=300, seed=0, interleaved=False):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.vocab = heads, kv_heads, dim, page, vocab
        self.interleaved = interleaved
        normal = lambda *shape: torch.randn(*shape, device=DEV, generator=self.g)
        # queries and keys in one tensor, as columns of a projection
        self.embedding = normal(vocab, heads + 2 * kv_heads, dim).to(torch.bfloat16)
        self.norm = 1 + 0.1 * normal(dim)
        self.head = normal(heads * dim, vocab) * 0.2
        self.frequencies, self.amplitude = smx.rotary_frequencies(dim, 1e4, scaling="yarn", factor=4.0, original_context=64)
        self.frequencies = self.frequencies.to(DEV)
        pages = requests * width
        self.k, self.v = (torch.zeros(pages, page, kv_heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.weights = torch.full((pages, kv_heads, page), float("nan"), device=DEV)  # (own keys start from zero)
        self.tables = torch.randperm(pages, device=DEV, generator=self.g).to(torch.int32).view(requests, width)
        self.context, self.positions = i32([0] * requests), i32([0] * requests)

    def step(self, tokens, new, max_new):
        """The new tokens (the last padding) through the layer; probabilities of the tokens behind them."""
        plan = smx.paged_plan(self.context, new, self.tables, page_size=self.page, num_pages=self.k.shape[0], tokens=len(tokens),
                              max_new=max_new)
        parts = self.embedding[tokens.clamp(0)]
        # a row's position: its request's, and its place in the step
        owner = torch.searchsorted(plan.starts.long(), torch.arange(len(tokens), device=DEV), right=True).sub(1).clamp(0, len(new) - 1)
        at = torch.where(plan.positions < 0, -1, plan.positions - self.context[owner] + self.positions[owner])
        rotated = smx.rotary(parts[:, :self.heads + self.kv_heads], at, self.frequencies, amplitude=self.amplitude, norm=self.norm,
                             interleaved=self.interleaved)
        query, key = rotated.split((self.heads, self.kv_heads), dim=1)
        smx.paged_write(key, parts[:, self.heads + self.kv_heads:], self.k, self.v, plan)
        lse = torch.empty(len(tokens), self.heads, device=DEV)
        out = smx.paged_attention(query, self.k, self.v, plan, lse=lse)
        smx.paged_key_weights(query, self.k, self.weights, plan, lse)
        probabilities = (out.flatten(1).float() @ self.head).softmax(1)
        return plan, at, rotated, out, probabilities


@pytest.mark.parametrize("interleaved,heads,kv_heads,dim", [(False, 8, 2, 64), (True, 3, 3, 128)])
def test_a_run_of_them_together(interleaved, heads, kv_heads, dim):
    requests, keep, recent, bound = 3, 40, 8, 56
    p = Program(requests, heads=heads, kv_heads=kv_heads, dim=dim, interleaved=interleaved, seed=dim)
    sim = [Request(kv_heads, dim) for _ in range(requests)]
    group, page = heads // kv_heads, p.page
    cpu = torch.Generator().manual_seed(1)
    emitted_before = [torch.randint(0, p.vocab, (n,), generator=cpu).tolist() for n in (50, 1, 9)]
    cuts = accepted = refused = 0
    for turn in range(14):
        # the tokens not yet in the cache, and drafts behind the last one
        drafts = [0 if turn == 0 else int(torch.randint(0, 4, (1,), generator=cpu)) for _ in range(requests)]
        if turn == 5:
            emitted_before[1] = []  # a request that pauses
            drafts[1] = 0
        count = [len(e) + d for e, d in zip(emitted_before, drafts)]
        total = sum(count) + 2
        # every draft from a distribution of its row: near enough to be accepted now and then
        draft = torch.randn(total, p.vocab, device=DEV, generator=p.g).mul(0.5).softmax(1)
        tokens, first = [], []
        for b in range(requests):
            first.append(len(tokens))
            row = emitted_before[b] + [0] * drafts[b]
            for i in range(drafts[b]):
                at = len(tokens) + len(emitted_before[b]) + i
                row[len(emitted_before[b]) + i] = int(torch.multinomial(draft[at - 1].cpu().double(), 1, generator=cpu))
            tokens += row
        tokens = torch.tensor(tokens + [0, 0], device=DEV)
        accept, sample = torch.rand(total, device=DEV, generator=p.g), torch.rand(requests, device=DEV, generator=p.g)
        before = p.weights.cpu().double()
        plan, at, rotated, out, target = p.step(tokens, i32(count), max(count))
        assert plan.status.tolist() == [smx.PAGED_OK] * requests

        # rotary: positions and values
        want_at = [s.position + i for s, c in zip(sim, count) for i in range(c)] + [-1, -1]
        assert at.tolist() == want_at
        inside = sum(count)
        parts = p.embedding[tokens][:inside, :heads + kv_heads]
        check(rotated[:inside], *rotate64(parts, at[:inside], p.frequencies, interleaved, p.amplitude, p.norm))
        assert rotated[inside:].eq(0).all()

        # attention and key weights, with the rotated heads as they are
        for b, s in enumerate(sim):
            rows = slice(first[b], first[b] + count[b])
            old = len(s.keys[0])
            q, key = rotated[rows].cpu().double().split((heads, kv_heads), dim=1)
            value = p.embedding[tokens[rows], heads + kv_heads:].cpu().double()
            table = p.tables[b].long().cpu()
            slots = lambda n: (table[torch.arange(n) // page], torch.arange(n) % page)
            for h in range(kv_heads):
                s.keys[h], s.values[h] = torch.cat((s.keys[h], key[:, h])), torch.cat((s.values[h], value[:, h]))
                n = len(s.keys[h])
                seen = torch.arange(n) <= old + torch.arange(count[b])[:, None]
                received = torch.cat((s.weights[h], torch.zeros(count[b], dtype=torch.float64)))
                for head in range(h * group, (h + 1) * group):
                    score = (q[:, head] @ s.keys[h].T / dim**0.5).masked_fill(~seen, -torch.inf)
                    weight = score.softmax(1)
                    got, exact = out[rows, head].cpu().double(), weight @ s.values[h]
                    # the result's rounding, the weights' to bf16 in the product and, where their sum is taken of the
                    # rounded ones, that; FP32 scores
                    size = weight @ s.values[h].abs()
                    assert ((got - exact).abs() <= 2**-7 * exact.abs() + (2**-8 + 2e-4) * size).all()
                    received += weight.sum(0)
                if count[b]:
                    page_of, slot_of = slots(n)
                    mine = p.weights.cpu().double()[page_of, h, slot_of]
                    assert not mine.isnan().any()
                    # exp of differences of FP32 scores (up to 128 products of size 1 / 8 and less) and sums of FP32
                    assert ((mine - received).abs() <= 2e-4 * received + 1e-9).all()
                    s.weights[h] = mine
        # pages of no request and slots behind the last key are left as they were
        untouched = torch.ones_like(p.weights, dtype=torch.bool).cpu()
        for b, s in enumerate(sim):
            n = len(s.keys[0])
            table = p.tables[b].long().cpu()
            untouched[table[torch.arange(n) // page], :, torch.arange(n) % page] = False
        assert torch.equal(p.weights.cpu().double()[untouched].nan_to_num(-1), before[untouched].nan_to_num(-1))

        # the drafts: verified rows are the last token and the drafts, of a plan of their own
        rows = [b for b in range(requests) for _ in range(1 + drafts[b] if count[b] else 0)]
        picked = torch.tensor([first[b] + count[b] - drafts[b] - 1 + i for b in range(requests) if count[b] for i in range(1 + drafts[b])],
                              device=DEV)
        verify_new = i32([1 + d if c else 0 for d, c in zip(drafts, count)])
        check_plan = smx.paged_plan(p.context * 0, verify_new, p.tables, page_size=page, num_pages=p.k.shape[0], tokens=len(rows))
        emitted, counts = smx.verify_drafts(target[picked], tokens[picked], check_plan, accept[picked], sample, draft=draft[picked])
        t64, d64 = target[picked].cpu().double(), draft[picked].cpu().double()
        at_row, next_tokens = 0, []
        for b in range(requests):
            if not count[b]:
                assert counts[b] == 0
                next_tokens.append([])
                continue
            mine, ids = [], tokens[picked].tolist()
            for i in range(drafts[b] + 1):
                row = at_row + i
                if i < drafts[b]:
                    x = ids[row + 1]
                    if accept[picked][row].item() * d64[row, x] < t64[row, x]:
                        mine.append(x)
                        accepted += 1
                        continue
                    refused += 1
                    left = (t64[row] - d64[row]).clamp(0)
                else:
                    left = t64[row]
                left = left if left.sum() > 0 else t64[row]
                sums = left.cumsum(0)
                mine.append(int((sums > sample[b].item() * sums[-1]).nonzero()[0]))
                break
            got = emitted[at_row:at_row + drafts[b] + 1].tolist()
            assert int(counts[b]) == len(mine) and got == mine + [-1] * (drafts[b] + 1 - len(mine))
            next_tokens.append(mine)
            at_row += drafts[b] + 1

        # the cache keeps the accepted tokens' keys; the drawn one comes with the next step
        for b, s in enumerate(sim):
            kept = count[b] - drafts[b] + max(0, len(next_tokens[b]) - 1)
            gone = count[b] - kept
            s.position += kept
            for h in range(kv_heads):
                n = len(s.keys[h]) - gone
                s.keys[h], s.values[h], s.weights[h] = s.keys[h][:n], s.values[h][:n], s.weights[h][:n]
            emitted_before[b] = next_tokens[b][-1:] if count[b] else torch.randint(0, p.vocab, (2,), generator=cpu).tolist()
        p.context, p.positions = i32([len(s.keys[0]) for s in sim]), i32([s.position for s in sim])

        # cut: requests over the bound, to `keep`
        goal = i32([keep if len(s.keys[0]) > bound - 12 else len(s.keys[0]) for s in sim])
        p.context = smx.paged_evict(p.k, p.v, p.weights, p.context, p.tables, goal, recent=recent)
        assert torch.equal(p.context, goal)
        for b, s in enumerate(sim):
            n, need = len(s.keys[0]), keep - recent
            if n > bound - 12:
                cuts += 1
                table = p.tables[b].long().cpu()
                for h in range(kv_heads):
                    order = torch.argsort(s.weights[h][:n - recent], descending=True, stable=True)
                    best = sorted(order[:need].tolist())
                    places = sorted(set(range(need)) - set(best))
                    index = list(range(need))
                    for place, source in zip(places, [i for i in best if i >= need]):
                        index[place] = source
                    index += list(range(n - recent, n))
                    s.keys[h], s.values[h], s.weights[h] = s.keys[h][index], s.values[h][index], s.weights[h][index]
            n = len(s.keys[0])
            table = p.tables[b].long().cpu()
            of, slot = table[torch.arange(n) // page], torch.arange(n) % page
            for h in range(kv_heads):
                assert torch.equal(p.k.cpu()[of, slot, h].double(), s.keys[h])
                assert torch.equal(p.v.cpu()[of, slot, h].double(), s.values[h])
                assert torch.equal(p.weights.cpu()[of, h, slot].double(), s.weights[h])
    assert cuts >= 3 and accepted >= 3 and refused >= 3  # (the run came to each)


def test_the_run_in_a_graph():
    """A whole turn, captured: each replay leaves what the same turn leaves eagerly."""
    def program():
        p = Program(4, width=10, seed=7)
        p.context.copy_(i32([60, 41, 3, 0])), p.positions.copy_(i32([900, 41, 3, 0]))
        p.k.normal_(generator=p.g), p.v.normal_(generator=p.g), p.weights.uniform_(generator=p.g)
        p.last, p.accept, p.sample = torch.zeros(4, 3, dtype=torch.long, device=DEV), torch.zeros(12, device=DEV), torch.zeros(4, device=DEV)
        p.new = i32([3, 3, 3, 3])
        return p

    def turn(p):
        tokens = p.last.flatten()
        plan, at, rotated, out, target = p.step(tokens, p.new, 3)
        emitted, counts = smx.verify_drafts(target, tokens, plan, p.accept, p.sample)
        p.context += counts
        p.positions += counts
        p.context.copy_(smx.paged_evict(p.k, p.v, p.weights, p.context, p.tables, 48, recent=10))
        return emitted, counts

    captured, eager = program(), program()
    turn(program())  # (loads every kernel)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = turn(captured)
    for p in (captured, eager):
        fresh = program()
        for name in ("context", "positions", "k", "v", "weights"):
            getattr(p, name).copy_(getattr(fresh, name))
    g = torch.Generator(device=DEV).manual_seed(8)
    for _ in range(12):
        last = torch.randint(0, eager.vocab, (4, 3), device=DEV, generator=g)
        accept, sample = torch.rand(12, device=DEV, generator=g) * 0.02, torch.rand(4, device=DEV, generator=g)
        for p in (captured, eager):
            p.last.copy_(last), p.accept.copy_(accept), p.sample.copy_(sample)
        want = turn(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(result, want):
            assert torch.equal(x, y)
        for name in ("context", "positions", "k", "v"):
            assert torch.equal(getattr(captured, name), getattr(eager, name)), name
        assert torch.equal(captured.weights.view(torch.int32), eager.weights.view(torch.int32))
    assert eager.context.max() <= 48 and eager.positions.max() > 900


def _pieces(block, x, *, positions=None, key_weights=None, tokens=80):
    """Three sequences through a block in pieces, as a serving loop runs them."""
    page, pages, width, length = 16, 40, 16, x.shape[1]
    k, v = (torch.zeros(pages, page, DIMS.kv_heads, DIMS.head_dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    weights = torch.full((pages, DIMS.kv_heads, page), float("nan"), device=DEV) if key_weights else None
    context, tables = i32([0] * 3), torch.randperm(pages, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    tables = tables[:3 * 12].view(3, 12).to(torch.int32)
    at, got = [0, 0, 0], [[], [], []]
    for new in ([33, 0, 5], [4, 40, 10], [10, 7, 17], [1, 1, 1], [0, 0, 15]):
        hidden = torch.zeros(tokens, DIMS.hidden, dtype=torch.bfloat16, device=DEV)
        hidden[:sum(new)] = torch.cat([x[b, at[b]:at[b] + n] for b, n in enumerate(new)])
        plan = smx.paged_plan(context, i32(new), tables, page_size=page, num_pages=pages, tokens=tokens, max_new=max(new))
        out = qb.block_step(hidden, block, k, v, plan, positions=positions(plan) if positions else None, key_weights=weights)
        for b, part in enumerate(out[:sum(new)].split(new)):
            got[b].append(part)
        context += plan.rows
        at = [a + n for a, n in zip(at, new)]
    assert at == [length] * 3
    return torch.stack([torch.cat(parts) for parts in got]), weights, tables


@pytest.mark.parametrize("arm", qb.SERVING_ARMS)
def test_block_steps_at_given_positions(arm):
    """Positions given, angles given, and both: the results of the tables, and the weights that every row's heads share out."""
    weights = qb.BlockWeights.random_init(DIMS, DEV, seed=1)
    make = lambda w=weights, **kw: qb.ServingBlock(w, DIMS, arm, max_context=256, tile=TILE, **kw)
    length, g = 48, torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(3, length, DIMS.hidden, device=DEV, generator=g).to(torch.bfloat16)
    plain = make()
    want, _, _ = _pieces(plain, x)
    given, received, tables = _pieces(plain, x, positions=lambda plan: plan.positions.long(), key_weights=True)
    # Both forms are within 2e-2 of the whole sequences' 64-bit block together (a bf16 rounding behind every operation); they
    # differ in the rotation alone, whose tables are FP32.
    assert (given.float() - want.float()).norm() <= 2e-2 * want.float().norm()
    # every row's heads share out 1 each; FP32 scores of normalised heads, 11.3 at most, each of 128 products
    for b in range(3):
        mine = received[tables[b].long()].transpose(1, 2).flatten(0, 1)
        group = DIMS.heads // DIMS.kv_heads
        assert (mine[:length].double().sum(0) - group * length).abs().max() <= 2e-4 * group * length
        assert mine[length:].isnan().all()
    # angles a fourth, positions four times: the same to the bit, since both factors are powers of two
    quarter = make(frequencies=plain.frequencies / 4)
    fourfold, _, _ = _pieces(quarter, x, positions=lambda plan: plan.positions * 4)
    assert torch.equal(fourfold, given)
    # without positions, the steps' own
    own, _, _ = _pieces(make(frequencies=plain.frequencies), x)
    assert torch.equal(own, given)
    # an amplitude of 2 takes back norms of a half
    halved = dataclasses.replace(weights, query_norm=weights.query_norm / 2, key_norm=weights.key_norm / 2)
    doubled, _, _ = _pieces(make(halved, frequencies=plain.frequencies, amplitude=2.0), x)
    assert torch.equal(doubled, given)
    with pytest.raises(ValueError, match="amplitude"):
        make(amplitude=2.0)


def test_another_stream():
    """The operators on a stream that is not the default one, with work before and behind them."""
    p = Program(2, seed=3)
    q = Program(2, seed=3)
    tokens = torch.arange(40, device=DEV)
    turn = lambda p: (p.step(tokens, i32([30, 10]), 30), smx.paged_evict(p.k, p.v, p.weights, i32([30, 10]), p.tables, 20, recent=4))
    want = turn(p)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = turn(q)
    stream.synchronize()
    assert torch.equal(got[1], want[1]) and torch.equal(got[0][3], want[0][3])
    assert torch.equal(p.k, q.k) and torch.equal(p.v, q.v)
    assert torch.equal(p.weights.view(torch.int32), q.weights.view(torch.int32))
