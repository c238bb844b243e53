"""Eviction of requests one of whose table entries is no page of the cache, wherever it lies: left as they were, their
lengths returned, nothing written through the entry."""

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_evict import check, make_cache
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("entry", [-1, "pages", 2**31 - 1])
@pytest.mark.parametrize("token", [2048, 4031, 20000, 33900])
@pytest.mark.parametrize("keep,recent", [(4096, 4096), (4096, 5000), (4096, 100), (0, 0)])
def test_entries_behind_those_read_first(keep, recent, token, entry):
    """More older tokens than sixteen waves hold, of which the waves' first 2048 each are read before the others: also where nothing
    survives for its weight, so that the weights themselves are not asked for. More heads and requests than go in parts."""
    page, context = 64, [38000, 38000] + [20] * 127
    k, v, weights, lens, tables = make_cache(context, page=page, kv_heads=1, seed=30)
    tables[0, token // page] = k.shape[0] if entry == "pages" else entry
    check((k, v, weights, lens, tables), context, keep, recent)


@pytest.mark.parametrize("keep,recent", [(5000, 5000), (5000, 300)])
@pytest.mark.parametrize("token", [0, 2100, 3500, 20000, 64990, 65010, 69999])
def test_entries_of_tables_wider_than_the_parts(keep, recent, token):
    page, context = 64, [70000, 900]
    k, v, weights, lens, tables = make_cache(context, page=page, kv_heads=2, seed=31, width=10000)
    tables[0, token // page] = -1
    check((k, v, weights, lens, tables), context, keep, recent)


@pytest.mark.parametrize("keep,recent", [(5000, 5000), (5000, 300)])
def test_entries_of_contexts_in_parts(keep, recent):
    page, context = 64, [70000, 70000, 70000, 70000, 900]
    k, v, weights, lens, tables = make_cache(context, page=page, kv_heads=2, seed=32)
    for b, token in enumerate((2100, 20000, 69999)):
        tables[b, token // page] = k.shape[0]
    check((k, v, weights, lens, tables), context, keep, recent)


def test_left_alone_and_cut_when_the_page_is_there():
    """The same request twice: with an entry missing it stays, with the entry it is cut."""
    page, context = 64, [40000] + [20] * 128
    k, v, weights, lens, tables = make_cache(context, page=page, kv_heads=1, seed=33)
    entry = tables[0, 2100 // page].clone()
    tables[0, 2100 // page] = -1
    before = [x.clone() for x in (k, v, weights)]
    assert smx.paged_evict(k, v, weights, lens, tables, 4096, recent=4096).tolist() == context[:1] + [20] * 128
    assert all(torch.equal(x, y) for x, y in zip((k, v, weights), before))
    tables[0, 2100 // page] = entry
    check((k, v, weights, lens, tables), context, 4096, 4096)
