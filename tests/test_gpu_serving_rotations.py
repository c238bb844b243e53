"""How far the two rotations of a serving step lie apart: by the block's tables (``paged_write``) and by positions (``rotary``)."""

import pytest
import torch

import strassen_tpu_amd as smx
from strassen_tpu_amd import qwen3_block as qb
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dim,theta", [(128, 1e6), (64, 1e4)])
@pytest.mark.parametrize("first", [0, 1000, 99_900])
def test_a_sequence_that_changes_from_tables_to_positions(dim, theta, first):
    """Heads at the same positions, near and far, by either: as near each other as the documentation of ``ServingBlock`` says."""
    tokens, page, heads = 96, 16, 2
    g = torch.Generator(device=DEV).manual_seed(60)
    k = torch.randn(tokens, heads, dim, device=DEV, generator=g).to(torch.bfloat16)
    context = torch.tensor([first], dtype=torch.int32, device=DEV)
    new = torch.tensor([tokens], dtype=torch.int32, device=DEV)
    pages = -(-(first + tokens) // page)
    cache = [torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    tables = torch.arange(pages, dtype=torch.int32, device=DEV)[None].contiguous()
    plan = smx.paged_plan(context, new, tables, page_size=page, num_pages=pages, tokens=tokens)
    cos, sin = qb.rope_values(first + tokens, dim, theta, DEV)
    if cos.shape[0] < plan.max_context:  # (a table for every position that the pages hold)
        cos, sin = qb.rope_values(plan.max_context, dim, theta, DEV)
    by_table = smx.paged_write(k, k, *cache, plan, q=k, rope_cos=cos, rope_sin=sin)
    f, _ = smx.rotary_frequencies(dim, theta, device=DEV)
    by_position = smx.rotary(k, plan.positions, f)
    # The angle: a power within four half steps of FP32 (2^-22 relative), its reciprocal and the product with the position (2^-24 each;
    # the exponents are exact for these head widths): below 2^-21. cos and sin: that, and a bf16 rounding (2^-8). A result of either path is rounded to bf16 once, and is
    # at most the sum of the pair; the FP32 arithmetic between is within one more part in a hundred of that.
    angle = (plan.positions.double()[:, None] * f * 2.0**-21)[:, None]
    both = k.double().abs()[..., :dim // 2] + k.double().abs()[..., dim // 2:]
    bound = (both * (angle + 2**-8) + 1.01 * 2 * 2**-8 * both).repeat(1, 1, 2)
    apart = (by_table.double() - by_position.double()).abs()
    assert (apart <= bound).all(), (apart / bound).max()
    if first == 0:  # at position 0 nothing is turned
        assert torch.equal(by_table[0], k[0]) and torch.equal(by_position[0], k[0])
