"""What verify_drafts reads stays as it was, and a request's tokens are the same in calls of other sizes."""

import ctypes

import pytest
import torch

import strassen_tpu_amd as smx
from strassen_tpu_amd import _lib
from test_gpu_parity import DEV, say
from test_gpu_verify import distributions, drawn, make_plan

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("vocab", [1000, 32001])  # a workgroup a request, and shared out
def test_inputs_stay_as_they_were(vocab, model):
    g = torch.Generator(device=DEV).manual_seed(70)
    new = [3, 0, 5, 1]
    target, draft = distributions(g, 10, vocab, torch.float32)
    tokens = drawn(g, draft)
    accept, sample = torch.rand(10, device=DEV, generator=g), torch.rand(4, device=DEV, generator=g)
    plan = make_plan(new, 10)
    read = [target, tokens, accept, sample, plan.starts, plan.rows, plan.context, plan.positions] + [draft] * model
    before, versions = [x.clone() for x in read], [x._version for x in read]
    smx.verify_drafts(target, tokens, plan, accept, sample, draft=draft if model else None)
    assert all(torch.equal(x, y) for x, y in zip(read, before)) and [x._version for x in read] == versions


def test_a_request_in_calls_of_other_sizes():
    """Alone (shared out over workgroups) and among 199 others (a workgroup each): the sums go in another order, and no random number
    of these lies so near a border that it shows."""
    g = torch.Generator(device=DEV).manual_seed(71)
    vocab, new = 32001, [3, 2]
    target, draft = distributions(g, 5, vocab, torch.float32)
    tokens = drawn(g, draft)
    accept, sample = torch.rand(5, device=DEV, generator=g), torch.rand(2, device=DEV, generator=g)
    # A sum of 32,001 values in any order is off by at most 32,000 roundings of 2^-53, 2^-38 of the whole. Borders further from the
    # number that is drawn with than both calls' sums and this loop's are off together (2^-36) decide alike in every order.
    for row in range(5):
        for p in (target[row].double(), (target[row].double() - draft[row].double()).clamp(min=0)):
            sums = p.cumsum(0)
            for u in sample.double():
                assert ((sums - u * sums[-1]).abs() > 2**-36 * sums[-1]).all()
    alone = [x.tolist() for x in smx.verify_drafts(target, tokens, make_plan(new), accept, sample, draft=draft)]
    many = lambda x, n: x.repeat((n,) + (1,) * (x.dim() - 1))
    got, counts = smx.verify_drafts(many(target, 100), many(tokens, 100), make_plan(new * 100), many(accept, 100), many(sample, 100),
                                    draft=many(draft, 100))
    assert got.tolist() == alone[0] * 100 and counts.tolist() == alone[1] * 100


@pytest.mark.parametrize("vocab", [1000, 32001])
def test_the_c_entry_reads_three_lists_of_a_step(vocab):
    """No tables, no stride and no contexts are asked for; results behind the lists that are read."""
    g = torch.Generator(device=DEV).manual_seed(72)
    new = [3, 0, 5, 1]
    target, draft = distributions(g, 9, vocab, torch.float32)
    tokens = drawn(g, draft).to(torch.int32)
    accept, sample = torch.rand(9, device=DEV, generator=g), torch.rand(4, device=DEV, generator=g)
    plan = make_plan(new)
    want = smx.verify_drafts(target, tokens, plan, accept, sample, draft=draft)
    lists = torch.cat((plan.starts[:4], plan.rows, plan.positions, torch.zeros(9 + 4, dtype=torch.int32, device=DEV)))
    starts, rows, positions, out, counts = lists.split((4, 4, 9, 9, 4))
    at = lambda x: x.data_ptr()
    step = _lib.SmxPagedStep(4, 9, 0, None, 0, at(starts), at(rows), None, at(positions))
    need = ctypes.c_int64()
    assert _lib.load().smx_verify_workspace_bytes(4, vocab, ctypes.byref(need)) == _lib.SMX_OK
    workspace = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    rc = _lib.load().smx_verify_drafts(ctypes.byref(step), vocab, at(target), vocab, at(draft), vocab, at(tokens), at(accept), at(sample), 0,
                                       at(out), at(counts), at(workspace), need.value, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.SMX_OK, _lib.last_error()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(counts, want[1])
