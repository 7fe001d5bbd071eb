"""Split counts of ragged 4-bit launches in small tiles, read back from the workspaces that the plan asks for: a long
request keeps its splits however many short ones share the launch."""
from __future__ import annotations

import ctypes

import pytest

from compactattention_amd import _hip
from tests.test_kv4_cpu import _dims, _ints


def _splits(need, rows):
    assert need == 0 or (need - 16) % (rows * 129 * 4) == 0
    return (need - 16) // (rows * 129 * 4) if need else 1


@pytest.mark.parametrize("heads,q_len,kv,least", [
    *(((32, 8), 1, [131072] + [640] * n, 16) for n in (7, 23, 29, 30, 31, 32, 47, 63)),
    ((32, 8), 1, [640] * 31 + [131072], 16), ((8, 8), 1, [64] * 40 + [60000] + [64] * 23, 16), ((9, 9), 1, [60000] + [64] * 63, 16),
    # drafts in tiles of 32 rows
    ((32, 8), 40, [131072] + [640] * 4, 4), ((32, 8), 40, [131072] + [640] * 7, 4), ((32, 8), 40, [131072] + [640] * 30, 4),
])
def test_decode(heads, q_len, kv, least):
    d = _dims(batch=len(kv), q_len=q_len, num_q_heads=heads[0], num_kv_heads=heads[1], kv_cap=-(-max(kv) // 64))
    need = _hip.lib().ca_attn_decode_q4_workspace_size(ctypes.byref(d), _ints(*kv), 0)
    assert _splits(need, len(kv) * heads[0] * q_len) >= least


@pytest.mark.parametrize("heads,chunk,past,least", [
    ((32, 8), 40, [2000] + [10] * 3, 4), ((32, 8), 40, [2000] + [10] * 5, 4), ((32, 8), 40, [10] * 20 + [2000], 4),
    ((16, 2), 20, [5, 900, 0, 60] + [1] * 20, 8),
])
def test_chunks(heads, chunk, past, least):
    d = _dims(batch=len(past), q_len=chunk, num_q_heads=heads[0], num_kv_heads=heads[1], kv_cap=max(past) + 1)
    need = _hip.lib().ca_attn_fwd_q4_workspace_size(ctypes.byref(d), _ints(*past), 0)
    assert _splits(need, len(past) * heads[0] * chunk) >= least


@pytest.mark.parametrize("kv,expect", [
    ([4096] * 32, 1), ([4000 + 3 * b for b in range(32)], 1),  # near even: a round of whole requests
    ([640] * 63 + [900], 1), ([254, 31001, 2047, 9000, 16385, 640, 23110, 4999], 10),
])
def test_even_requests_as_before(kv, expect):
    d = _dims(batch=len(kv), q_len=1, num_q_heads=32, num_kv_heads=8, kv_cap=-(-max(kv) // 64))
    need = _hip.lib().ca_attn_decode_q4_workspace_size(ctypes.byref(d), _ints(*kv), 0)
    assert _splits(need, len(kv) * 32) == expect
