"""Rows of a serving step through a whole block: what lies in the rows of no admitted request stays there."""

import math

import pytest
import torch

import strassen_tpu_amd as smx
import strassen_tpu_amd.qwen3_block as qb
from test_gpu_parity import DEV, say
from test_gpu_serving_block import DIMS, TILE, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("value", [0.0, 3e38, math.inf, math.nan])
@pytest.mark.parametrize("arm", qb.SERVING_ARMS)
def test_rows_of_no_request_do_not_reach_others(arm, value):
    """Padding rows and rows of a request that is not admitted, uninitialised memory as far as the step is concerned: the
    admitted rows and the cache get the same bits whatever they hold."""
    weights = qb.BlockWeights.random_init(DIMS, DEV, seed=1)
    block = qb.ServingBlock(weights, DIMS, arm, max_context=64, tile=TILE)
    new, tokens = [7, 9, 3], 48  # the second breaks max_new
    rows = torch.randn(tokens, DIMS.hidden, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(torch.bfloat16)
    admitted = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    admitted[:7], admitted[16:19] = True, True

    def step(x):
        k, v = (torch.zeros(8, 16, DIMS.kv_heads, DIMS.head_dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        plan = smx.paged_plan(i32([0, 0, 5]), i32(new), i32([[0, -1], [1, -1], [2, -1]]), page_size=16, num_pages=8,
                              tokens=tokens, max_new=8, max_context=32)
        assert plan.status.tolist() == [smx.PAGED_OK, smx.PAGED_BAD_LENGTH, smx.PAGED_OK]
        return qb.block_step(x, block, k, v, plan), k, v

    want = step(torch.where(admitted[:, None], rows, 0))
    x = torch.where(admitted[:, None], rows, value)
    kept = x.clone()
    got = step(x)
    assert want[0][admitted].isfinite().all()
    assert torch.equal(got[0][admitted], want[0][admitted])
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
    assert torch.equal(x.nan_to_num(7.0), kept.nan_to_num(7.0))  # the step's input stays
