"""Results of rotary, attention's row sums, key weights and eviction over what the same call reads beside them: refused before any
launch."""

import pytest

from strassen_tpu_amd import _lib
from test_serving_operators import FAR, OUT, _evict, _key_weights, _rotary, _verify, refused
from test_serving_surface import P, _cache, _heads, _step


# eight rows of eight heads of 128: 16384 bytes of bf16, 32768 of float32
@pytest.mark.parametrize("change", [
    dict(positions=OUT), dict(positions=OUT + 16380), dict(positions=OUT - 28), dict(positions=OUT - 56, flags=8),
    dict(frequencies=OUT + 16376), dict(frequencies=OUT - 504), dict(frequencies=OUT - 252, flags=4),
    dict(norm=OUT + 16382), dict(norm=OUT - 254), dict(norm=OUT - 508, flags=2), dict(norm=OUT + 32764, flags=3),
    # in place
    dict(x=_heads(data=OUT), positions=OUT + 64), dict(x=_heads(data=OUT), norm=OUT + 64),
])
def test_rotary_refuses_results_over_what_it_reads(change):
    refused(_rotary(**change), "positions, frequencies and norm")


# eight pages of two heads of 16 slots: 1024 bytes; two requests, eight tokens, tables of four entries
@pytest.mark.parametrize("change", [
    dict(starts=FAR), dict(starts=FAR + 1020), dict(starts=FAR - 4), dict(rows=FAR + 512), dict(rows=FAR - 4), dict(context=FAR),
    dict(context=FAR + 1020), dict(positions=FAR - 28), dict(positions=FAR + 1020), dict(tables=FAR), dict(tables=FAR + 1020),
    dict(tables=FAR - 16),
])
def test_key_weights_refuse_weights_over_the_steps_lists(change):
    refused(_key_weights(step=_step(**change)), "step's lists")


# eight pages of sixteen rows of two heads of 128: 65536 bytes of keys, as many of values 2^24 behind them, 1024 of weights
@pytest.mark.parametrize("base,size", [(OUT, 65536), (OUT + (1 << 24), 65536), (FAR, 1024)])
@pytest.mark.parametrize("change", [
    dict(context=0), dict(context=-4), dict(lens=-4), dict(keep_lens=-4), dict(tables=-28), dict(tables=-4), dict(context="end"),
    dict(lens="end"), dict(keep_lens="end"), dict(tables="end"),
])
def test_evict_refuses_rows_and_weights_over_the_lists(base, size, change):
    apart = dict(context=1 << 20, tables=1 << 21, lens=1 << 22)
    refused(_evict(**{**apart, **{name: base + (size - 4 if at == "end" else at) for name, at in change.items()}}),
            "lengths and block_tables")


# eight rows of eight heads: 256 bytes
@pytest.mark.parametrize("change", [
    dict(starts=FAR), dict(starts=FAR + 252), dict(rows=FAR - 4), dict(context=FAR + 128), dict(positions=FAR - 28),
    dict(positions=FAR + 252), dict(tables=FAR + 252), dict(tables=FAR - 16),
])
def test_attention_refuses_row_sums_over_the_steps_lists(change):
    refused(_lib.load().smx_paged_attention_lse(_cache(k=OUT, v=OUT + (1 << 24)), _step(**change), _heads(data=1 << 30),
                                                _heads(data=1 << 30), 0.1, 0, 0, FAR, P, 0, None), "step's lists")


# eight rows of 100 probabilities, two requests: `out` of 32 bytes at OUT (64 of int64), `counts` of 8 at FAR
@pytest.mark.parametrize("change", [
    dict(counts=OUT), dict(counts=OUT + 28), dict(counts=OUT + 60, flags=2), dict(counts=OUT - 4), dict(accept=OUT - 28), dict(accept=FAR + 4),
    dict(sample=OUT + 28), dict(sample=FAR - 4), dict(tokens=FAR - 28), dict(tokens=FAR - 56, flags=2), dict(target=OUT + 28),
    dict(target=OUT - 4 * (700 + 100) + 4), dict(target=FAR - 4 * (7 * 128 + 100) + 4, target_row=128), dict(draft=OUT + 28, draft_row=100),
    dict(draft=FAR - 2 * 800 + 4, draft_row=100, flags=1), dict(step=_step(starts=FAR)), dict(step=_step(rows=FAR)),
    dict(step=_step(rows=OUT + 28)), dict(step=_step(positions=FAR - 28)), dict(step=_step(positions=OUT)),
])
def test_verify_refuses_results_over_what_it_reads(change):
    refused(_verify(**{**dict(out=OUT, counts=FAR), **change}), "share no memory")
