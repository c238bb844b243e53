"""Verification of drafted tokens on the GPU against a loop in 64 bits."""

import math

import numpy as np
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


def make_plan(new, tokens=None, max_new=None):
    lens = torch.zeros(len(new), dtype=torch.int32, device=DEV)
    width = -(-max(max(new), 1) // 16)
    tables = torch.arange(len(new) * width, dtype=torch.int32, device=DEV).view(len(new), width)
    return smx.paged_plan(lens, torch.tensor(new, dtype=torch.int32, device=DEV), tables, page_size=16,
                          num_pages=len(new) * width, tokens=tokens or max(1, sum(new)), max_new=max_new)


def expected(target, tokens, new, accept, sample, draft, count):
    """One request after another, in numpy's 64 bits."""
    clean = lambda x: np.where((x > 0) & (x < np.inf), x, 0.0)
    target, draft = clean(target.double().cpu().numpy()), None if draft is None else clean(draft.double().cpu().numpy())
    tokens, accept, sample = tokens.tolist(), accept.double().tolist(), sample.double().tolist()
    out, counts, start, vocab = [-1] * count, [], 0, target.shape[1]
    for b, n in enumerate(new):
        if not n:
            counts.append(0)
            continue
        a = 0
        while a < n - 1:
            x, row = tokens[start + a + 1], start + a
            p = target[row, x] if 0 <= x < vocab else 0.0
            q = 1.0 if draft is None else draft[row, x] if 0 <= x < vocab else 0.0
            if not (p > 0 and accept[row] * q < p):
                break
            out[start + a] = x
            a += 1
        rest = target[start + a].copy()
        if a < n - 1:
            if draft is not None:
                rest = np.maximum(rest - draft[start + a], 0)
            elif 0 <= tokens[start + a + 1] < vocab:
                rest[tokens[start + a + 1]] = 0
            if not rest.sum() > 0:
                rest = target[start + a].copy()
        sums = rest.cumsum()
        fits = np.nonzero((sums > sample[b] * sums[-1]) & (rest > 0))[0]
        held = np.nonzero(rest > 0)[0]
        out[start + a] = int(fits[0]) if len(fits) else int(held[-1]) if len(held) else -1
        counts.append(a + 1)
        start += n
    return out, counts


def distributions(g, rows, vocab, dtype, noise=0.7, spread=3.0):
    logits = spread * torch.randn(rows, vocab, device=DEV, generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    return target, torch.softmax(logits + noise * torch.randn(rows, vocab, device=DEV, generator=g), -1).to(dtype)


def drawn(g, draft):
    """Tokens of a step: row i + 1 holds one drawn from row i's draft."""
    noise = torch.rand(draft.shape, device=DEV, generator=g).clamp_(min=1e-9)
    return torch.roll((draft.float() / -noise.log()).argmax(-1), 1)


def check(new, vocab, dtype=torch.float32, *, model=True, pad=0, tokens_dtype=torch.int64, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + vocab)
    rows = sum(new) + pad
    target, draft = distributions(g, rows, vocab, dtype)
    tokens = drawn(g, draft).to(tokens_dtype)
    accept, sample = torch.rand(rows, device=DEV, generator=g), torch.rand(len(new), device=DEV, generator=g)
    plan = make_plan(new, rows)
    got, counts = smx.verify_drafts(target, tokens, plan, accept, sample, draft=draft if model else None)
    want, want_counts = expected(target, tokens, new, accept, sample, draft if model else None, rows)
    assert got.dtype == tokens_dtype and counts.dtype == torch.int32
    assert counts.tolist() == want_counts and got.tolist() == want
    return want_counts


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new,vocab", [
    ([1], 151936), ([5], 151936), ([1, 3, 0, 7, 2], 32001), ([4] * 30, 1000), ([2, 0, 9], 4096), ([3, 3], 4097), ([200, 1, 70], 513),
    ([3], 1), ([2, 4], 2), ([1] * 300, 77),
])
def test_verify(new, vocab, dtype, model):
    counts = check(new, vocab, dtype, model=model, pad=3)
    if new == [4] * 30 and model:
        assert {1, 4} < set(counts)  # some refused at once, some taken whole


@pytest.mark.parametrize("requests,vocab,dtype,model", [
    # a workgroup a request, of 512 threads and of 1024, and requests shared out, on both sides of each border
    (3, 4096, torch.float32, True), (3, 4097, torch.float32, True), (3, 8192, torch.bfloat16, False), (3, 8193, torch.bfloat16, True),
    (191, 9001, torch.bfloat16, False), (192, 9001, torch.bfloat16, False), (256, 8001, torch.float32, True),
    (257, 8001, torch.float32, True), (512, 65536, torch.bfloat16, False), (260, 65537, torch.bfloat16, False),
    (513, 300, torch.float32, True), (200, 32001, torch.float32, True), (700, 2049, torch.bfloat16, False)])
def test_requests_whole_and_shared_out(requests, vocab, dtype, model):
    check([(7 * b + 1) % 4 for b in range(requests)], vocab, dtype, model=model, pad=5)


def test_vocabulary_of_more_slices_than_threads():
    check([3, 1], 4_500_001, tokens_dtype=torch.int32)


def test_many_rounds():
    for seed in range(12):
        check([1 + (seed + b) % 6 for b in range(64)], 1500 + 37 * seed, seed=seed, pad=seed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_on_the_borders(dtype):
    """Eighths, whose sums and products are exact: numbers that meet a border fall to the token behind it, and an
    acceptance number that meets the quotient refuses."""
    vocab = 64
    p, q = torch.zeros(2, vocab, device=DEV, dtype=dtype), torch.zeros(2, vocab, device=DEV, dtype=dtype)
    p[:, [3, 10, 11, 40]] = torch.tensor([0.25, 0.25, 0.375, 0.125], device=DEV, dtype=dtype)
    q[:, [3, 10, 40, 60]] = torch.tensor([0.5, 0.125, 0.25, 0.125], device=DEV, dtype=dtype)
    plan, sure = make_plan([2]), torch.tensor([0.0], device=DEV)

    def run(token, accept, sample, draft=q):
        tokens = torch.tensor([7, token], device=DEV)
        got, counts = smx.verify_drafts(p, tokens, plan, torch.tensor([accept, 0.0], device=DEV), torch.tensor([sample], device=DEV), draft=draft)
        return got[:int(counts)].tolist()

    # p / q of token 3 is a half
    assert run(3, 0.5 - 2**-25, 0.0) == [3, 3] and run(3, 0.5, 0.0) == [10]
    # max(p - q, 0): 10 has an eighth, 11 three
    assert [run(3, 0.75, u) for u in (0.0, 0.25 - 2**-26, 0.25, 1 - 2**-24, 1.0, 2.0, math.nan)] == [[10], [10], [11], [11], [11], [11], [11]]
    # all of p behind an accepted draft
    assert [run(10, 0.9, u)[1] for u in (0.0, 0.25 - 2**-26, 0.25, 0.5, 0.875 - 2**-24, 0.875, 1.0)] == [3, 3, 10, 11, 11, 40, 40]
    # not drawn: accepted by p alone, the refused one left out
    # (0.375 - 2**-26 lies half way between two float32 numbers and becomes 0.375, which refuses)
    assert run(11, 0.375 - 2**-25, 0.0, None) == [11, 3] and run(11, 0.375 - 2**-26, 0.0, None) == [3]
    assert [run(11, 0.375, u, None) for u in (0.39, 0.4, 0.8)] == [[3], [10], [40]]
    # tokens without probability, or outside the vocabulary
    assert run(60, 0.0, 0.0) == [10] and run(5, 0.0, 0.0, None) == [3]
    for outside in (-1, vocab, 2**40, -2**40):
        assert run(outside, 0.0, 0.5) == [11] and run(outside, -1.0, 0.5, None) == [11]
    assert sure.item() == 0


def test_rows_that_leave_nothing():
    """p below q everywhere: from p; no probability at all: -1; values that are none count as zero."""
    vocab = 5000
    p, q = torch.zeros(2, vocab, device=DEV), torch.zeros(2, vocab, device=DEV)
    p[:, [100, 4500]] = 0.25
    q[:, [100, 4500]] = 0.5
    tokens, accept = torch.tensor([0, 100], device=DEV), torch.tensor([0.9, 0.0], device=DEV)
    plan = make_plan([2])
    run = lambda p, q, u: [x.tolist() for x in smx.verify_drafts(p, tokens, plan, accept, torch.tensor([u], device=DEV), draft=q)]
    assert run(p, q, 0.1) == [[100, -1], [1]] and run(p, q, 0.6) == [[4500, -1], [1]]
    assert run(torch.zeros_like(p), q, 0.6) == [[-1, -1], [1]]
    p[:, [7, 8, 9]], q[:, 4500] = torch.tensor([math.nan, math.inf, -1.0], device=DEV), math.nan
    assert run(p, q, 0.1) == [[4500, -1], [1]]
    only = torch.zeros(2, vocab, device=DEV)
    only[:, 100] = 0.5  # refused though it is all there is: from p, without it nothing is left
    assert run(only, None, 0.3) == [[100, -1], [1]]


def test_probabilities_in_views():
    """Padded vocabularies, rows of a larger tensor, repeated and transposed rows."""
    g = torch.Generator(device=DEV).manual_seed(8)
    new, vocab = [3, 1, 4], 999
    target, draft = distributions(g, 8, vocab, torch.float32)
    tokens = drawn(g, draft)
    accept, sample = torch.rand(8, 2, device=DEV, generator=g)[:, 0], torch.rand(3, 5, device=DEV, generator=g)[:, 1]
    plan = make_plan(new, 8)
    want = [x.tolist() for x in smx.verify_drafts(target, tokens, plan, accept.contiguous(), sample.contiguous(), draft=draft)]
    assert want[0] == expected(target, tokens, new, accept, sample, draft, 8)[0]
    padded = torch.full((8, vocab + 25), 9.0, device=DEV)
    padded[:, :vocab] = target
    for p, q in ((padded[:, :vocab], draft), (target.t().contiguous().t(), draft.t().contiguous().t())):
        assert [x.tolist() for x in smx.verify_drafts(p, torch.stack((tokens, tokens), 1)[:, 0], plan, accept, sample, draft=q)] == want
    one = target[:1].expand(8, vocab)
    got, _ = smx.verify_drafts(one, tokens, plan, accept, sample, draft=draft)
    assert got.tolist() == expected(one, tokens, new, accept, sample, draft, 8)[0]


def test_requests_that_are_not_admitted():
    g = torch.Generator(device=DEV).manual_seed(9)
    new, vocab = [2, 6, 3], 300
    target, draft = distributions(g, 11, vocab, torch.float32)
    tokens, accept, sample = drawn(g, draft), torch.rand(11, device=DEV, generator=g), torch.rand(3, device=DEV, generator=g)
    whole = smx.verify_drafts(target, tokens, make_plan(new, 11), accept, sample, draft=draft)
    some = smx.verify_drafts(target, tokens, make_plan(new, 11, max_new=4), accept, sample, draft=draft)
    assert some[1].tolist() == [whole[1][0].item(), 0, whole[1][2].item()]
    assert torch.equal(some[0][:2], whole[0][:2]) and torch.equal(some[0][8:], whole[0][8:]) and (some[0][2:8] == -1).all()


def test_emitted_tokens_follow_the_target():
    """What is emitted first is distributed as the target's first row, whatever the drafts: 200,000 requests' worth of
    numbers. A share of m draws is off by at most 5 sqrt(p (1 - p) / m) but once in two million."""
    g = torch.Generator(device=DEV).manual_seed(10)
    vocab, requests, rounds = 6, 2000, 100
    p, q = (torch.softmax(torch.randn(vocab, device=DEV, generator=g), -1) for _ in range(2))
    plan, seen = make_plan([2] * requests), torch.zeros(vocab, device=DEV, dtype=torch.int64)
    target, draft = p.expand(2 * requests, vocab).contiguous(), q.expand(2 * requests, vocab).contiguous()
    for _ in range(rounds):
        tokens = torch.multinomial(q, 2 * requests, replacement=True, generator=g)
        accept, sample = torch.rand(2 * requests, device=DEV, generator=g), torch.rand(requests, device=DEV, generator=g)
        got, counts = smx.verify_drafts(target, tokens, plan, accept, sample, draft=draft)
        seen += torch.bincount(got[0::2], minlength=vocab)
    share, m = seen.double() / (requests * rounds), requests * rounds
    assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / m).sqrt()).all()


def test_in_a_graph():
    g = torch.Generator(device=DEV).manual_seed(11)
    new = torch.tensor([3, 1, 5, 0], dtype=torch.int32, device=DEV)
    lens, tables = torch.zeros_like(new), torch.arange(4, dtype=torch.int32, device=DEV)[:, None].contiguous()
    target, draft = distributions(g, 16, 5000, torch.float32)
    tokens, accept, sample = drawn(g, draft), torch.rand(16, device=DEV, generator=g), torch.rand(4, device=DEV, generator=g)

    def step():
        plan = smx.paged_plan(lens, new, tables, page_size=16, num_pages=4, tokens=16)
        return smx.verify_drafts(target, tokens, plan, accept, sample, draft=draft)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        emitted, counts = step()
    for i in range(4):
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(emitted, want[0]) and torch.equal(counts, want[1])
        new.copy_(torch.tensor([[0, 7, 1, 2], [16, 0, 0, 0], [4, 4, 4, 4], [1, 1, 1, 1]][i]))
        accept.copy_(torch.rand(16, device=DEV, generator=g)), sample.copy_(torch.rand(4, device=DEV, generator=g))


def test_refusals():
    plan = make_plan([2, 1])
    target, tokens = torch.rand(3, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    accept, sample = torch.rand(3, device=DEV), torch.rand(2, device=DEV)
    for change, message in (
            (dict(target=target[:2]), "target"), (dict(target=target.half()), "target"), (dict(target=target[0]), "target"),
            (dict(target=target[:, :0]), "target"), (dict(tokens=tokens[:2]), "tokens"), (dict(tokens=tokens.float()), "tokens"),
            (dict(accept=accept[:2]), "accept"), (dict(accept=accept.double()), "accept"), (dict(sample=accept), "sample"),
            (dict(draft=target[:, :7]), "draft"), (dict(draft=target.to(torch.bfloat16)), "draft"), (dict(draft=target.cpu()), "HIP device"),
            (dict(target=target.clone().requires_grad_()), "gradients")):
        args = {"target": target, "tokens": tokens, "plan": plan, "accept": accept, "sample": sample, **change}
        with pytest.raises(ValueError, match=message):
            smx.verify_drafts(args.pop("target"), args.pop("tokens"), args.pop("plan"), args.pop("accept"), args.pop("sample"), **args)
