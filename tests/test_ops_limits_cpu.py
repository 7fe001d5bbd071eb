"""Host arguments beyond what the C interface holds are refused, not taken modulo 2^32."""
from __future__ import annotations

import pytest

from compactattention_amd import ops


@pytest.mark.parametrize("value", [1 << 31, (1 << 32) + 5, -(1 << 31) - 1, 1 << 70])
def test_per_request_values_fit_32_bits(value):
    for vals in ([value], [1, value], [value, 0, 7]):
        with pytest.raises(ValueError, match="32 bits"):
            ops.past_array(vals)
        with pytest.raises(ValueError, match="32 bits"):
            ops.past_array(vals, len(vals))
        with pytest.raises(ValueError, match="32 bits"):
            ops.attn_decode_workspace_bytes(vals, 1, 8, 2, 1 << 20)
    with pytest.raises(ValueError, match="32 bits"):
        ops._starts(value, 2, 1)


def test_per_request_values_at_the_edges():
    vals = [-(1 << 31), 0, (1 << 31) - 1]
    assert list(ops.past_array(vals, 3)) == vals
