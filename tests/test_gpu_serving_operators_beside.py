"""Operands of the serving operators that lie back to back in one allocation, as a program's own arena holds them."""

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_evict import expected, make_cache, same
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def arena(*parts):
    """Copies of the tensors behind each other, each where the one before ends (sizes are multiples of 16 bytes)."""
    memory = torch.empty(sum(x.numel() * x.element_size() for x in parts), dtype=torch.uint8, device=DEV)
    views, at = [], 0
    for x in parts:
        size = x.numel() * x.element_size()
        assert size % 16 == 0
        views.append(memory[at:at + size].view(x.dtype).view(x.shape).copy_(x))
        at += size
    return views


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (1, 0, 2, 3), (2, 1, 0, 3), (3, 2, 1, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_beside_what_it_reads(dtype, order):
    g = torch.Generator(device=DEV).manual_seed(50)
    x = torch.randn(16, 8, 128, device=DEV, generator=g).to(dtype)
    positions = torch.randint(0, 5000, (16,), device=DEV, generator=g, dtype=torch.int32)
    f = smx.rotary_frequencies(128, device=DEV)[0]
    norm = torch.randn(128, device=DEV, generator=g).to(dtype)
    want = smx.rotary(x, positions, f, norm=norm)
    parts = [torch.zeros_like(x), positions, f, norm]
    laid = arena(*(parts[i] for i in order))
    out, positions, f, norm = (laid[order.index(i)] for i in range(4))
    assert smx.rotary(x, positions, f, norm=norm, out=out) is out
    assert torch.equal(out, want)
    out.copy_(x)  # in place
    assert torch.equal(smx.rotary(out, positions, f, norm=norm, out=out), want)
    with pytest.raises(ValueError, match="positions, frequencies and norm"):
        smx.rotary(x, out.view(torch.int32).flatten()[:16], f, out=out)


@pytest.mark.parametrize("max_new", [1, 40])
def test_key_weights_beside_the_steps_lists(max_new):
    """Weights between the tables and the lengths, the plan made from both."""
    g = torch.Generator(device=DEV).manual_seed(51)
    k = torch.randn(12, 16, 2, 128, device=DEV, generator=g).to(torch.bfloat16)
    q = torch.randn(4 * max_new, 4, 128, device=DEV, generator=g).to(torch.bfloat16)
    tables = torch.randperm(12, device=DEV, generator=g)[:12].view(4, 3).to(torch.int32)
    lens, new = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 5, 7, 8], [max_new] * 4))
    first = torch.rand(12, 2, 16, device=DEV, generator=g)

    def run(tables, weights, lens, lse):
        plan = smx.paged_plan(lens, new, tables, page_size=16, num_pages=12, tokens=4 * max_new, max_new=max_new)
        smx.paged_attention(q, k, k, plan, lse=lse)
        smx.paged_key_weights(q, k, weights, plan, lse)
        return weights, lse

    lse = torch.zeros(4 * max_new, 4, device=DEV)
    want = run(tables, first.clone(), lens, lse)
    got = run(*arena(tables, first, lens, lse))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_eviction_beside_the_lists():
    """Keys, lengths, values, tables and weights one behind the other."""
    context, keep = [100, 30, 65, 77], [40, 40, 8, 70]
    k, v, w, lens, tables = make_cache(context, page=8, seed=52, width=16)
    want = expected(k, v, w, context, tables, keep, 6)
    goals = torch.tensor(keep, dtype=torch.int32, device=DEV)
    k, lens, v, tables, w, goals = arena(k, lens, v, tables, w, goals)
    assert smx.paged_evict(k, v, w, lens, tables, goals, recent=6).tolist() == want[3] and lens.tolist() == context
    assert same(k, want[0]) and same(v, want[1]) and same(w, want[2])
    with pytest.raises(ValueError, match="lengths and block_tables"):
        smx.paged_evict(k, v, w, w.view(torch.int32).flatten()[:4], tables, goals, recent=6)
