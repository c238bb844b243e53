"""Eviction from long contexts whose weights follow the keys' order, as those do that keys have received from the rows behind them."""

import pytest
import torch

from test_gpu_evict import check, make_cache
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("context,keep,recent", [([131000], 32768, 512), ([131000, 40003], 4096, 100), ([524288], 3001, 0)])
@pytest.mark.parametrize("kind", ["falling", "falling and noisy", "rising", "steps"])
def test_weights_along_a_long_context(context, keep, recent, kind):
    k, v, w, lens, tables = make_cache(context, page=64, kv_heads=1, seed=40)
    g = torch.Generator(device=DEV).manual_seed(41)
    for b, n in enumerate(context):
        at = torch.arange(n, device=DEV)
        fall = torch.log(n / (at + 1).double()) + 1 / n  # every row shares out 1 among the keys before it
        if kind == "falling and noisy":
            fall = fall * (0.5 * torch.randn(n, device=DEV, generator=g)).exp()
        elif kind == "rising":
            fall = (at + 1).double()
        elif kind == "steps":  # of which each sampled key may be the only one
            fall = torch.exp2(-(at // 997).double() % 100)
        w[tables[b].long()[at // 64], 0, at % 64] = fall.float()
    check((k, v, w, lens, tables), context, keep, recent)
