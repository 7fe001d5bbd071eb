"""Arguments beyond what the C interface or a launch holds are refused before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from compactattention_amd import _hip, ops
from tests.test_kv4_cpu import FAKE, INVALID, LIMIT, _dims, _ints, _kv4, _seq


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


@pytest.mark.parametrize("batch,heads,length,code", [
    (1, 1 << 10, 1 << 18, LIMIT), (64, 1 << 4, 1 << 18, LIMIT), (1, 1, 1 << 28, LIMIT), (1, 1, (1 << 28) - 15, LIMIT),
    (64, (1 << 31) - 1, (1 << 31) - 1, LIMIT), (1, 1, (1 << 28) - 16, INVALID), (3, 5, 17895696, INVALID),
])
def test_rows_of_a_launch(batch, heads, length, code):
    """16 threads a row: 2^28 rows would be 2^32 threads.  (INVALID: the start, which is looked at after the rows.)"""
    lib, d, kv, s = _hip.lib(), _dims(batch=batch, q_len=length, num_kv_heads=heads, kv_cap=1 << 24), _kv4(pts=1 << 25), _seq()
    r = [ctypes.byref(x) for x in (d, s, kv)]
    start = _ints(*([-1] * batch))
    assert lib.ca_append_q4(r[0], r[1], r[1], r[2], r[2], start, None) == code
    assert lib.ca_gather_q4(r[0], r[2], r[2], start, FAKE, FAKE, None) == code


@pytest.mark.parametrize("page_bytes,pages,code", [(2048, (1 << 25) - 1, LIMIT), (2048, (1 << 25) - 2, INVALID), (1 << 22, 1 << 14, LIMIT),
                                                   (1 << 22, (1 << 14) - 1, INVALID)])
def test_bytes_of_a_copy(page_bytes, pages, code):
    """16 bytes a thread, rounded up to workgroups of 256.  (INVALID: every id is 0, which is looked at afterwards.)"""
    pool = (_hip.PagePool * 1)(_hip.PagePool(FAKE, page_bytes, page_bytes, 1 << 26))
    ids = np.zeros(pages, np.int32)
    assert _hip.lib().ca_copy_pages(pool, 1, ids.ctypes.data, ids.ctypes.data, pages, None, None) == code
