"""NaN in queries, keys and values of a 4-bit cache comes through every way in which splits are joined: few rows, many
rows of few splits, many rows of many splits, whatever the split that holds it weighs."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd import ops
from tests.test_gpu_kv4 import SCALE, _check, _lists, _poison, _tables
from tests.test_gpu_kv4_sizes import _big_cache, _q

pytestmark = pytest.mark.gpu

CHUNKS = [
    # (Hq, Hkv, chunk, past blocks, splits): tiles of 32 rows, then of 256; splits of few and of more than 4096 rows
    (16, 2, 300, 100, 2), (16, 2, 300, 100, 6), (8, 2, 64, 100, 7), (16, 16, 300, 100, 3), (16, 16, 300, 100, 6),
    (16, 16, 200, 200, 16), (32, 8, 256, 128, 0),
]


@pytest.mark.parametrize("Hq,H,L,past,splits", CHUNKS)
def test_chunks(gpu, Hq, H, L, past, splits):
    print(f"case: kv4 nan chunk heads={Hq}/{H} chunk={L} past={past} splits={splits}", flush=True)
    G, qb = Hq // H, -(-L // 64)
    cap = past + qb
    K, V, kt, vt = _big_cache(H, cap, gpu, seed=L)
    lists = _lists(1, H, [past], qb, 0.7, seed=past)
    last = past + (L - 1) // 64
    lists[0][1] = [last]  # one block, so one split alone has keys
    first = lists[0][0][0]
    _poison(K, V, kt, vt, 0, 64 * first + 5, {"k": [1]})  # a key that every query of the row sees
    _poison(K, V, kt, vt, 1, 64 * past + L - 2, {"k": [3]})  # the last two queries see it, in their only block
    q = _q(gpu, 1, L, Hq, 128, seed=1)
    q[0, L // 2, G + G - 1, 77] = float("nan")  # a query that sees no key stays at zeros
    q[0, L - 3, G, 0] = float("nan")
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, [past], SCALE, cap, H, with_lse=True, num_splits=splits)
    assert torch.isnan(out[0, :, :G]).all() and torch.isnan(lse[0, :G]).all()
    assert torch.isnan(out[0, L - 2:, G:2 * G]).all() and torch.isnan(lse[0, G:2 * G, L - 2:]).all()
    assert torch.isnan(out[0, L - 3, G]).all() and torch.isnan(lse[0, G, L - 3])
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * past], [64 * past + L])


@pytest.mark.parametrize("Hq,H,L,lens,splits", [(8, 2, 1, [2000], 6), (32, 8, 16, [3000, 700], 5), (64, 4, 64, [6405, 7680], 6)])
def test_tokens_and_drafts(gpu, Hq, H, L, lens, splits):
    print(f"case: kv4 nan decode heads={Hq}/{H} q_len={L} lens={lens} splits={splits}", flush=True)
    blocks = -(-max(lens) // 64)
    K, V, kt, vt = _big_cache(len(lens) * H, blocks, gpu, seed=L)
    q = _q(gpu, len(lens), L, Hq, 128, seed=2)
    q[0, L - 1, 0, 9] = float("nan")
    _poison(K, V, kt, vt, 1, lens[0] - 1, {"k": [0]})  # the last query alone
    out, lse = ops.attn_decode(q, K, V, lens, SCALE, blocks, H, with_lse=True, num_splits=splits)
    G = Hq // H
    assert torch.isnan(out[0, L - 1, :1]).all() and torch.isnan(lse[0, 0, L - 1])
    assert torch.isnan(out[0, L - 1, G:2 * G]).all() and torch.isfinite(out[0, :L - 1]).all()
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)


@pytest.mark.parametrize("Hq,H,L,past,splits", [(8, 8, 1, 12, 3), (16, 2, 300, 100, 2), (16, 2, 300, 100, 6), (8, 2, 64, 100, 7),
                                                (16, 16, 300, 100, 6)])
def test_values_in_a_split_of_no_weight(gpu, Hq, H, L, past, splits):
    """Scores of -181 in the first blocks and 181 in the rest: the first split's weight is 0 in fp32, and a NaN value in
    it is a NaN sum all the same, as it is without splits."""
    print(f"case: kv4 nan value of no weight heads={Hq}/{H} q_len={L} past={past} splits={splits}", flush=True)
    qb = -(-L // 64)
    cap = past + qb
    K, V, kt, vt = _big_cache(H, cap, gpu, seed=5)
    cut = -(-cap // splits)  # the first split's blocks
    plus, minus = 0x66, 0xEE  # two codes of 4 and of -4, under a scale of 1
    K.tensor[:, :4096] = plus
    K.tensor[:, 4096:] = 127
    low = kt[:, :cut].reshape(-1).long().to(gpu)
    K.tensor[low, :4096] = minus
    q = torch.full((1, L, Hq, 128), 4.0, dtype=torch.bfloat16, device=gpu)
    for h in range(H):
        _poison(K, V, kt, vt, h, 7, {"v": [h % 4]})
    n = 64 * past + L
    lists = [[list(range(cap))] * H]
    if L == 1:
        out, lse = ops.attn_decode(q, K, V, [n], SCALE, cap, H, with_lse=True, num_splits=splits)
    else:
        table, counts = _tables(lists, cap, gpu)
        out, lse = ops.attn_fwd(q, K, V, table, counts, [past], SCALE, cap, H, with_lse=True, num_splits=splits)
    G = Hq // H
    for h in range(H):
        o = out[0, :, h * G:(h + 1) * G].unflatten(-1, (4, 32))
        assert torch.isnan(o[..., h % 4, :]).all() and torch.isfinite(o[..., (h + 1) % 4, :]).all()
    assert torch.isfinite(lse).all()
