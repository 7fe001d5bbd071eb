"""Block tables of a 4-bit cache with entries outside the request's blocks."""
from __future__ import annotations

import pytest

from compactattention_amd import ops
from tests.test_gpu_kv4 import SCALE, _cache, _check, _tables
from tests.test_gpu_kv4_sizes import _q

pytestmark = pytest.mark.gpu


def test_list_ids_past_the_last_block(gpu):
    """An id past the request's last block is that block, wherever in the list it stands."""
    print("case: chunk4 ids past the last block", flush=True)
    for H, Hq, L, past in ((2, 8, 150, 20), (16, 16, 300, 100)):
        qb = -(-L // 64)
        cap = past + qb
        K, V, kt, vt = _cache(1, H, cap, gpu, seed=9)
        q = _q(gpu, 1, L, Hq, 128)
        ids = [3, past, past + 1, 7, cap - 1]
        for at, splits in ((4, 1), (4, 2), (1, 1), (0, 1)):
            row = ids[:4]
            row.insert(at, cap - 1)
            lists = [[row] * H]
            table, counts = _tables(lists, cap, gpu)
            table[:, at] = (1 << 29) + 5
            out, lse = ops.attn_fwd(q, K, V, table, counts, [past], SCALE, cap, H, with_lse=True, num_splits=splits)
            _check(out, lse, q, K, V, kt, vt, H, lists, [64 * past], [64 * past + L], every=5)
