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


@pytest.mark.parametrize("a,b,fine", [
    # (offset, page bytes, stride, pages) twice
    ((0, 4352, 4352, 100), (435200, 4352, 4352, 100), True), ((0, 4352, 4352, 100), (435184, 4352, 4352, 100), False),
    ((0, 4352, 4352, 100), (0, 4352, 4352, 100), True),    # one pool, named twice
    ((0, 4352, 4352, 100), (0, 4352, 4352, 50), True),
    ((0, 4352, 4352, 100), (4352, 4352, 4352, 100), False),  # the same pages under other ids
    ((0, 4352, 8704, 100), (4352, 4352, 8704, 100), True),   # K and V in turn
    ((4352, 4352, 8704, 100), (0, 4352, 8704, 100), True), ((0, 4352, 8704, 100), (4336, 4352, 8704, 100), False),
    ((0, 4352, 8704, 100), (4368, 4352, 8704, 100), False), ((0, 1024, 4096, 10), (2048, 1024, 8192, 10), True),
    ((0, 1024, 4096, 10), (8192, 1024, 8192, 10), False), ((0, 1024, 1024, 100), (0, 2048, 2048, 50), False),
    ((0, 1024, 1024, 1 << 40), (1 << 50, 1024, 1024, 1 << 60), True), ((0, 1024, 1024, 1 << 60), (1 << 50, 1024, 2048, 8), False),
])
def test_pools_of_a_copy_do_not_overlap(a, b, fine):
    """A page of one pool that another pool knows by another id could be read and written in one call."""
    pools = (_hip.PagePool * 3)(*(_hip.PagePool(FAKE + p[0], *p[1:]) for p in (a, b, (16 - FAKE, 16, 16, 1))))
    lib = _hip.lib()
    assert lib.ca_copy_pages(pools, 3, None, None, 0, None, None) == (0 if fine else INVALID)
    swapped = (_hip.PagePool * 2)(pools[1], pools[0])
    assert lib.ca_copy_pages(swapped, 2, None, None, 0, None, None) == (0 if fine else INVALID)
    assert fine or "overlap" in _hip.last_error()
