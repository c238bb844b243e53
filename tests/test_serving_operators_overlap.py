"""Results of rotary, attention's row sums, key weights and eviction over what the same call reads beside them: refused before any
launch."""

import pytest

from test_serving_operators import OUT, _rotary, refused
from test_serving_surface import _heads


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
