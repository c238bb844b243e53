"""The decoder block as a serving step: prompts in pieces and decoded tokens over a
paged cache give what the block gives on whole sequences."""

import pytest
import torch

import strassen_tpu_amd as smx
import strassen_tpu_amd.qwen3_block as qb
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu

DIMS = qb.Qwen3Dims(hidden=512, ffn=1024, heads=8, kv_heads=2)
TILE = (256, 256)


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Server:
    """A cache, its free pages and the requests' lengths, as a serving loop keeps them."""

    def __init__(self, block, requests, tokens, page=16, pages=40, width=16):
        self.block, self.tokens, self.page = block, tokens, page
        self.k, self.v = (torch.zeros(pages, page, DIMS.kv_heads, DIMS.head_dim, dtype=torch.bfloat16, device=DEV)
                          for _ in range(2))
        self.context = i32([0] * requests)
        self.tables = i32([[-1] * width] * requests)
        self.free = torch.randperm(pages, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9)).to(torch.int32)

    def step(self, rows, max_new=None):
        """``rows``: each request's new hidden states. Returns the requests' results."""
        new = [r.shape[0] for r in rows]
        x = torch.zeros(self.tokens, DIMS.hidden, dtype=torch.bfloat16, device=DEV)
        x[:sum(new)] = torch.cat(rows)
        plan = smx.paged_plan(self.context, i32(new), self.tables, page_size=self.page, num_pages=self.k.shape[0],
                              tokens=self.tokens, free_pages=self.free, max_new=max_new)
        out = qb.block_step(x, self.block, self.k, self.v, plan)
        assert plan.status.tolist() == [smx.PAGED_OK] * len(rows)
        self.context += plan.rows
        self.free = self.free[int(plan.pages_used):].contiguous()
        return out[:sum(new)].split(new)


def dequantised(weights, group=128):
    """The weights that the 4-bit arm computes with (to bf16's rounding)."""
    def back(w):
        codes, scales, zeros = smx.int4_quantize(w, group)
        spread = lambda t: t.float().repeat_interleave(group, 0)
        return ((codes.float() - spread(zeros)) * spread(scales)).to(torch.bfloat16)

    names = ("query", "key", "value", "attention_output", "gate_up", "mlp_down")
    return qb.dataclasses.replace(weights, **{n: back(getattr(weights, n)) for n in names})


@pytest.mark.parametrize("arm", qb.SERVING_ARMS)
def test_steps_give_whole_sequences(arm):
    weights = qb.BlockWeights.random_init(DIMS, DEV, seed=1)
    block = qb.ServingBlock(weights, DIMS, arm, max_context=256, tile=TILE)
    length, g = 48, torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(3, length, DIMS.hidden, device=DEV, generator=g).to(torch.bfloat16)
    whole = qb.PreparedBlock(dequantised(weights) if arm == "int4" else weights, DIMS, "hipblaslt", batch=3, seq=length)
    want = qb.block_forward(x.flatten(0, 1), whole).view(3, length, -1)

    server, at, got = Server(block, 3, 80), [0, 0, 0], [[], [], []]
    # prompts in pieces, then tokens one by one, requests coming and going
    for new in ([33, 0, 5], [4, 40, 10], [10, 7, 17], [1, 1, 1], [0, 0, 15]):
        rows = [x[b, at[b]:at[b] + n] for b, n in enumerate(new)]
        for b, out in enumerate(server.step(rows, max_new=1 if max(new) == 1 else None)):
            got[b].append(out)
        at = [a + n for a, n in zip(at, new)]
    assert at == [length] * 3
    got = torch.stack([torch.cat(parts) for parts in got])
    assert got.isfinite().all()
    # The block's products, norms and attention follow one another with a bf16 rounding each, in both
    # forms: 9e-3 from the 64-bit block is what its GEMM arms have, twice that for two of them.
    assert (got.float() - want.float()).norm() <= 2e-2 * want.float().norm()


def test_step_in_a_graph():
    """A decode step, captured once: each replay gives the eager step's bits."""
    weights = qb.BlockWeights.random_init(DIMS, DEV, seed=3)
    for arm in qb.SERVING_ARMS:
        block = qb.ServingBlock(weights, DIMS, arm, max_context=256, tile=TILE)
        g = torch.Generator(device=DEV).manual_seed(4)
        server = Server(block, 16, 16, pages=64, width=4)
        server.step([torch.randn(n, DIMS.hidden, device=DEV, generator=g).to(torch.bfloat16) for n in (1,) * 16])
        x = torch.randn(16, DIMS.hidden, device=DEV, generator=g).to(torch.bfloat16)
        context, new, free = server.context.clone(), i32([1] * 16), server.free.clone()

        def step():
            plan = smx.paged_plan(context, new, server.tables, page_size=16, num_pages=64, tokens=16, free_pages=free,
                                  max_new=1)
            return qb.block_step(x, block, server.k, server.v, plan), plan

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, plan = step()
        for _ in range(3):
            want, eager = step()
            kept = want.clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, kept), arm
            context += eager.rows
            x.copy_(torch.randn(16, DIMS.hidden, device=DEV, generator=g))


def test_serving_block_refusals():
    weights = qb.BlockWeights.random_init(DIMS, DEV, seed=5)
    with pytest.raises(ValueError, match="unknown arm"):
        qb.ServingBlock(weights, DIMS, "hipblaslt", max_context=64)
    block = qb.ServingBlock(weights, DIMS, "int4", max_context=64)
    server = Server(block, 1, 16)  # tables of 256 positions, RoPE tables of 64
    with pytest.raises(ValueError, match="positions"):
        server.step([torch.zeros(1, DIMS.hidden, dtype=torch.bfloat16, device=DEV)])
