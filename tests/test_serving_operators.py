"""Rotary positions, key weights, eviction and verification of drafts: what needs no GPU. Refusals of the C entry
points before any launch, refusals of tensors that the calls cannot take, and the angles of the rotations."""

import ctypes
import math
import os
import re

import pytest
import torch

import strassen_tpu_amd as smx
from strassen_tpu_amd import _lib
from test_serving_surface import BAD_CACHES, P, _cache, _heads, _step

FAR, OUT = 1 << 32, 1 << 31  # aligned addresses that no refused call reads


def test_constants_match_the_header():
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                               "strassen_mi355x.h")).read()
    for name in ("SMX_ROTARY_F32", "SMX_ROTARY_NORM_F32", "SMX_ROTARY_FREQUENCIES_F32", "SMX_ROTARY_POSITIONS_I64",
                 "SMX_ROTARY_INTERLEAVED", "SMX_VERIFY_BF16", "SMX_VERIFY_TOKENS_I64"):
        assert int(re.search(rf"#define {name} (\d+)", header).group(1)) == getattr(_lib, name)
    assert re.search(r"#define SMX_VERIFY_MAX_VOCAB \(1 << (\d+)\)", header).group(1) == "28"
    assert _lib.SMX_VERIFY_MAX_VOCAB == 1 << 28


def refused(rc, message):
    said = _lib.last_error()
    assert rc in (_lib.SMX_ERR_INVALID, _lib.SMX_ERR_UNSUPPORTED) and message in said, (rc, said)


def _rotary(tokens=8, head_dim=128, rotary_dim=128, x=None, out=None, positions=P, frequencies=P, norm=None, flags=0,
            amplitude=1.0, eps=1e-6, zero_rows=0):
    return _lib.load().smx_rotary(tokens, head_dim, rotary_dim, x or _heads(data=FAR), out or _heads(data=OUT), positions,
                                  frequencies, norm, flags, amplitude, eps, zero_rows, None)


@pytest.mark.parametrize("change,message", [
    (dict(tokens=0), "tokens"), (dict(tokens=(1 << 20) + 1), "tokens"), (dict(x=_heads(0, data=FAR)), "heads"),
    (dict(x=_heads(65536, data=FAR), out=_heads(65536, data=OUT)), "heads"), (dict(out=_heads(4, data=OUT)), "as many"),
    (dict(x=_heads(data=None)), "null"), (dict(positions=None), "null"), (dict(frequencies=None), "null"),
    (dict(head_dim=1), "head_dim"), (dict(head_dim=1026), "head_dim"), (dict(rotary_dim=0), "rotated"),
    (dict(rotary_dim=63), "rotated"), (dict(rotary_dim=130), "rotated"), (dict(flags=32), "flags"), (dict(flags=-1), "flags"),
    (dict(amplitude=math.inf), "amplitude"), (dict(amplitude=math.nan), "amplitude"), (dict(eps=-1e-9), "eps"),
    (dict(eps=math.nan), "eps"), (dict(x=_heads(data=FAR + 1)), "misaligned"), (dict(x=_heads(data=FAR + 2), flags=1), "misaligned"),
    (dict(x=_heads(data=FAR, token=-1)), "negative"), (dict(positions=P + 2), "misaligned"),
    (dict(positions=P + 4, flags=8), "misaligned"), (dict(frequencies=P + 4), "misaligned"), (dict(norm=P + 1), "misaligned"),
    (dict(norm=P + 2, flags=2), "misaligned"),
    # rows of the result on each other; a result that meets the heads without being them
    (dict(out=_heads(data=OUT, token=0)), "each other"), (dict(out=_heads(data=OUT, token=7 * 128)), "each other"),
    (dict(out=_heads(data=OUT, head=64)), "each other"), (dict(out=_heads(data=FAR, token=2048)), "share no memory"),
    (dict(out=_heads(data=FAR + 2 * 128)), "share no memory"), (dict(x=_heads(data=OUT, token=0)), "share no memory"),
])
def test_rotary_refusals(change, message):
    refused(_rotary(**change), message)


def _verify(step=None, vocab=100, target=P, target_row=100, draft=None, draft_row=0, tokens=P, accept=P, sample=P, flags=0, out=P,
            counts=P, workspace=P, size=1 << 20):
    return _lib.load().smx_verify_drafts(step or _step(), vocab, target, target_row, draft, draft_row, tokens, accept, sample, flags,
                                         out, counts, workspace, size, None)


@pytest.mark.parametrize("change,message", [
    (dict(step=_step(requests=0)), "requests"), (dict(step=_step(requests=8193)), "requests"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 28) + 1), "vocab"), (dict(step=_step(tokens=0)), "tokens"), (dict(step=_step(tokens=(1 << 20) + 1)), "tokens"),
    (dict(step=_step(starts=None)), "null"), (dict(step=_step(rows=None)), "null"), (dict(step=_step(positions=None)), "null"),
    (dict(target=None), "null"), (dict(tokens=None), "null"), (dict(accept=None), "null"), (dict(sample=None), "null"),
    (dict(out=None), "null"), (dict(counts=None), "null"), (dict(flags=4), "flags"), (dict(target_row=99), "apart"),
    (dict(draft=P, draft_row=99), "apart"), (dict(target=P + 2), "misaligned"), (dict(target=P + 1, flags=1), "misaligned"),
    (dict(draft=P + 2, draft_row=100), "misaligned"), (dict(tokens=P + 4, flags=2), "misaligned"), (dict(out=P + 4, flags=2), "misaligned"),
    (dict(accept=P + 2), "misaligned"), (dict(sample=P + 1), "misaligned"), (dict(counts=P + 2), "misaligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=P + 8), "workspace"), (dict(size=16), "workspace"),
    (dict(out=P + 28), "share no memory"), (dict(tokens=P + 56, flags=2), "share no memory"),
])
def test_verify_refusals(change, message):
    refused(_verify(**change), message)


def _evict(cache=None, weights=FAR, requests=2, width=4, context=P, tables=P, stride=4, keep_lens=None, keep=8, recent=2,
           max_context=64, lens=P, workspace=P, size=1 << 20):
    return _lib.load().smx_paged_evict(cache or _cache(k=OUT, v=OUT + (1 << 24)), weights, requests, width, context, tables, stride,
                                       keep_lens, keep, recent, max_context, lens, workspace, size, None)


@pytest.mark.parametrize("change,message", [({"cache": _cache(**{"k": OUT, "v": OUT + (1 << 24), **c})}, "") for c in BAD_CACHES] + [
    (dict(requests=0), "requests"), (dict(requests=8193), "requests"), (dict(weights=None), "null"), (dict(context=None), "null"),
    (dict(tables=None), "null"), (dict(lens=None), "null"), (dict(keep=-1), "keep"), (dict(recent=-1), "recent"),
    (dict(width=0), "table_stride"), (dict(stride=3), "table_stride"), (dict(max_context=65), "max_context"),
    (dict(max_context=-1), "max_context"), (dict(max_context=(1 << 30) + 1), "max_context"), (dict(weights=FAR + 4), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=P + 4), "workspace"), (dict(size=15), "workspace"),
    # rows that meet: of the keys, of keys and values, of the weights and either
    (dict(cache=_cache(k=OUT, v=OUT + (1 << 24), page_stride=16 * 256 - 128)), "each other"),
    (dict(cache=_cache(k=OUT, v=OUT)), "keys and values"), (dict(cache=_cache(k=OUT, v=OUT + 256)), "keys and values"),
    (dict(weights=OUT + 1024), "key_weights must share"), (dict(weights=OUT + (1 << 24) - 16), "key_weights must share"),
    (dict(context=1 << 20, tables=1 << 21, lens=(1 << 20) + 4), "lens must share"), (dict(context=1 << 20, tables=1 << 21, lens=(1 << 21) + 28), "lens must share"),
    (dict(context=1 << 20, tables=1 << 21, keep_lens=P), "lens must share"),
])
def test_evict_refusals(change, message):
    refused(_evict(**change), message)


def test_evict_workspaces():
    """Of every bound on the contexts: enough for the lists of the rows that can move, and the same for the call."""
    bytes_ = ctypes.c_int64()

    def workspace(requests, heads, keep, most):
        assert _lib.load().smx_paged_evict_workspace_bytes(requests, heads, keep, most, ctypes.byref(bytes_)) == _lib.SMX_OK
        return bytes_.value

    for requests, heads, keep, most in ((1, 1, 0, 0), (1, 8, 100, 64), (4, 8, 32768, 131072), (64, 8, 2048, 8192), (3, 2, -1, 40000),
                                        (1, 1, 1000, 1 << 30), (8192, 8, 1, 100)):
        moves = most // 2 if keep < 0 else min(keep, max(0, most - keep))
        need = workspace(requests, heads, keep, most)
        assert need >= requests * heads * 8 * moves and need < (1 << 42)
    assert _lib.load().smx_paged_evict_workspace_bytes(1, 0, 1, 1, ctypes.byref(bytes_)) == _lib.SMX_ERR_INVALID
    assert _lib.load().smx_paged_evict_workspace_bytes(1, 1, 1, 1, None) == _lib.SMX_ERR_INVALID


def _key_weights(cache=None, step=None, q=None, lse=P, scale=0.1, window=0, weights=FAR, workspace=P, size=0):
    return _lib.load().smx_paged_key_weights(cache or _cache(k=OUT, v=OUT), step or _step(), q or _heads(data=1 << 30), lse, scale,
                                             window, weights, workspace, size, None)


@pytest.mark.parametrize("change,message", [({"cache": _cache(**c)}, "") for c in BAD_CACHES] + [
    (dict(step=_step(requests=0)), "requests"), (dict(step=_step(tokens=0)), "tokens"), (dict(step=_step(max_new=-1)), "step"),
    (dict(step=_step(tables=None)), "null"), (dict(step=_step(starts=None)), "null"), (dict(step=_step(rows=None)), "null"),
    (dict(step=_step(context=None)), "null"), (dict(lse=None), "null"), (dict(weights=None), "null"), (dict(q=_heads(data=None)), "null"),
    (dict(q=_heads(7, data=1 << 30)), "query heads"), (dict(q=_heads(0, data=1 << 30)), "query heads"),
    (dict(q=_heads(258, data=1 << 30)), "query heads"), (dict(q=_heads(data=(1 << 30) + 2)), "aligned"),
    (dict(q=_heads(data=1 << 30, token=1025)), "aligned"), (dict(q=_heads(data=1 << 30, head=-128)), "aligned"),
    (dict(q=_heads(data=1 << 30, token=1 << 28)), "2^32"), (dict(q=_heads(data=1 << 30, head=1 << 30)), "2^32"),
    (dict(q=_heads(data=1 << 30, token=1 << 40)), "2^32"), (dict(lse=P + 2), "misaligned"), (dict(weights=FAR + 4), "misaligned"),
    (dict(weights=OUT), "key_weights must share"), (dict(weights=(1 << 30) + 4096), "key_weights must share"),
    (dict(lse=FAR + 16), "key_weights must share"), (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=3e38), "scale"), (dict(scale=math.nan), "scale"), (dict(window=-1), "window"),
])
def test_key_weights_refusals(change, message):
    refused(_key_weights(**change), message)


def _calls(device="cpu"):
    """Each call with tensors whose types and shapes it takes."""
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=device)
    bf16 = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=device)
    yield lambda: smx.rotary(bf16(3, 2, 64), ints(3), torch.ones(32, dtype=torch.float64, device=device))
    yield lambda: smx.paged_evict(bf16(4, 16, 2, 64), bf16(4, 16, 2, 64), torch.zeros(4, 2, 16, device=device), ints(1), ints(1, 4), 3)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    for call in _calls():
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_fake_and_traced_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    with FakeTensorMode():
        for call in _calls("cuda"):
            with pytest.raises(ValueError, match="traced|plain strided tensor"):
                call()
    x, positions, frequencies = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), torch.ones(32)
    with pytest.raises(ValueError, match="traced"):
        make_fx(lambda x: smx.rotary(x, positions, frequencies))(x)
    with pytest.raises(ValueError, match="plain strided tensor|gradients"):
        torch.vmap(lambda x: smx.rotary(x, positions, frequencies))(x[None])


def test_plain_angles():
    for dim, theta in ((2, 1e4), (64, 1e6), (128, 10.0), (128, 0.5), (6, 1.0)):
        got, amplitude = smx.rotary_frequencies(dim, theta)
        assert got.dtype == torch.float64 and got.shape == (dim // 2,) and amplitude == 1.0
        # a power whose exponent is rounded once, and the function's own rounding
        want = torch.tensor([theta ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
        torch.testing.assert_close(got, want, rtol=2**-50 * (1 + abs(math.log(theta))), atol=0)


def test_stretched_angles():
    """Each scaling by what it says of the fastest, the slowest and every other pair."""
    dim, theta, factor, original = 128, 1e6, 8.0, 4096
    plain, _ = smx.rotary_frequencies(dim, theta)
    close = dict(rtol=1e-13, atol=0)
    got, amplitude = smx.rotary_frequencies(dim, theta, scaling="linear", factor=factor)
    torch.testing.assert_close(got * factor, plain, **close)
    assert amplitude == 1.0
    got, amplitude = smx.rotary_frequencies(dim, theta, scaling="ntk", factor=factor)
    assert amplitude == 1.0 and got[0] == 1.0
    torch.testing.assert_close(got[-1] * factor, plain[-1], **close)
    steps = got[1:] / got[:-1]  # a power of one base
    torch.testing.assert_close(steps, steps[:1].expand_as(steps), **close)
    assert smx.rotary_frequencies(2, theta, scaling="ntk", factor=factor)[0].tolist() == [1.0]

    turns = original * plain / (2 * math.pi)
    got, amplitude = smx.rotary_frequencies(dim, theta, scaling="bands", factor=factor, original_context=original)
    assert amplitude == 1.0
    for p, t, f in zip(plain.tolist(), turns.tolist(), got.tolist()):
        stays = min(1.0, max(0.0, (t - 1) / 3))
        assert f == pytest.approx(p * stays + p / factor * (1 - stays), rel=1e-13)
    assert (turns > 4).any() and (turns < 1).any() and ((turns > 1) & (turns < 4)).any()

    got, amplitude = smx.rotary_frequencies(dim, theta, scaling="yarn", factor=factor, original_context=original)
    assert amplitude == pytest.approx(1 + 0.1 * math.log(8), rel=1e-15)
    # the last pair that turns 32 times, the first that turns at most once
    low, high = int((turns >= 32).sum()) - 1, int((turns > 1).sum())
    assert 0 < low < high < dim // 2
    for i, (p, f) in enumerate(zip(plain.tolist(), got.tolist())):
        part = min(1.0, max(0.0, (i - low) / (high - low)))
        assert f == pytest.approx(p * (1 - part) + p / factor * part, rel=1e-13)
    same, amplitude = smx.rotary_frequencies(dim, theta, scaling="yarn", factor=1, original_context=original)
    torch.testing.assert_close(same, plain, **close)
    assert amplitude == 1.0


@pytest.mark.parametrize("args,message", [
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=63), "rotary_dim"), (dict(theta=0.0), "theta"), (dict(theta=math.inf), "theta"),
    (dict(factor=2.0), "scaling="), (dict(scaling="other"), "unknown"), (dict(scaling="linear", factor=0.5), "factor"),
    (dict(scaling="ntk", factor=math.nan), "factor"), (dict(scaling="yarn", factor=2.0), "original_context"),
    (dict(scaling="bands", factor=2.0, original_context=0), "original_context"),
    (dict(scaling="bands", factor=2.0, original_context=100, fast=1.0), "fast"),
    (dict(scaling="yarn", factor=2.0, original_context=100, slow=0.0), "slow"),
    (dict(scaling="yarn", factor=2.0, original_context=100, theta=1.0), "theta"),
])
def test_angles_refused(args, message):
    with pytest.raises(ValueError, match=message):
        smx.rotary_frequencies(**{"rotary_dim": 64, **args})
