"""Attention over a 4-bit cache at its edges: many KV rows, lists in any order, random shapes and splits, full lengths,
several streams at once."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from compactattention_amd import ops
from tests import kv4_oracle as ref
from tests.test_gpu_kv4 import SCALE, _cache, _check, _lists, _poison, _tables

pytestmark = pytest.mark.gpu


def _q(gpu, *shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(gpu)


def _big_cache(rows, blocks, gpu, seed):
    """Random pages made on the GPU: codes at random, scales 2^-8 .. 2^0, so values to 6."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    total = rows * blocks
    pools = []
    for _ in range(2):
        p = torch.randint(0, 256, (total, ref.PAGE), generator=g, device=gpu, dtype=torch.uint8)
        p[:, 4096:] = torch.randint(119, 128, (total, 256), generator=g, device=gpu, dtype=torch.uint8)
        pools.append(p)
    tables = [torch.randperm(total, generator=g, device=gpu).view(rows, blocks).to(torch.int32) for _ in range(2)]
    return *(ops.KV4.paged(p, t) for p, t in zip(pools, tables)), *(t.cpu() for t in tables)


@pytest.mark.parametrize("Hq,H,L", [(9, 9, 1), (18, 9, 12), (9, 9, 40)])
def test_more_rows_than_the_plan_places(gpu, Hq, H, L):
    """64 requests x 9 KV heads: 576 rows, past the 512 that the plan places one by one."""
    print(f"case: kv4 576 rows heads={Hq}/{H} q_len={L}", flush=True)
    B = 64
    lens = [L + (37 * b) % 300 for b in range(B)]
    blocks = -(-max(lens) // 64)
    K, V, kt, vt = _big_cache(B * H, blocks, gpu, seed=L)
    q = _q(gpu, B, L, Hq, 128)
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    for splits in (0, 2):
        out, lse = ops.attn_decode(q, K, V, lens, SCALE, blocks, H, with_lse=True, num_splits=splits)
        _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens, every=7)


def test_more_rows_than_the_plan_places_in_a_chunk(gpu):
    print("case: chunk4 576 rows", flush=True)
    B, H, Hq, L = 64, 9, 9, 70
    past = [b % 5 for b in range(B)]
    K, V, kt, vt = _big_cache(B * H, 6, gpu, seed=3)
    q = _q(gpu, B, L, Hq, 128)
    lists = _lists(B, H, past, 2, 0.6, seed=4)
    table, counts = _tables(lists, 6, gpu)
    for splits in (0, 2):
        out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, 6, H, with_lse=True, num_splits=splits)
        _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past], every=7)


@pytest.mark.parametrize("splits", [1, 3])
def test_lists_in_any_order_and_with_repeats(gpu, splits):
    """Blocks of a list in no order, the chunk's own first, one named twice (it counts twice), one past the request's
    last (read as the last)."""
    print(f"case: chunk4 unordered lists splits={splits}", flush=True)
    H, Hq, L, past = 2, 8, 150, [20]
    cap = 23
    K, V, kt, vt = _cache(1, H, cap, gpu, seed=9)
    rng = np.random.default_rng(5)
    a = [22, 21, 20] + rng.permutation(20).tolist()
    b = [3, 3, 21, 7, 20, 1, 22, 0, 19, 11, 21]
    lists = [[a, b]]
    table, counts = _tables(lists, cap, gpu)
    table[1, 4] = 1 << 29  # past the last block: the last block
    lists[0][1][4] = 22
    q = _q(gpu, 1, L, Hq, 128)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [1280], [1280 + L])


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(gpu, seed):
    rng = np.random.default_rng(1000 + seed)
    H = int(rng.integers(1, 6))
    G = int(rng.integers(1, 17))
    B = int(rng.integers(1, 5))
    if seed % 2:
        L = int(rng.integers(1, 65))
        lens = [L + int(rng.integers(0, 1500)) for _ in range(B)]
        blocks = -(-max(lens) // 64)
        splits = int(rng.choice([0, 0, 1, 2, 5, 33, 64]))
        print(f"case: kv4 random decode heads={G * H}/{H} q_len={L} lens={lens} splits={splits}", flush=True)
        K, V, kt, vt = _cache(B, H, blocks, gpu, seed=seed)
        q = _q(gpu, B, L, G * H, 128, seed=seed)
        out, lse = ops.attn_decode(q, K, V, lens, SCALE, blocks, H, with_lse=True, num_splits=splits)
        lists = [[list(range(-(-n // 64)))] * H for n in lens]
        _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)
        return
    L = int(rng.integers(1, 400))
    past = [int(rng.integers(0, 30)) for _ in range(B)]
    qb = -(-L // 64)
    cap = max(past) + qb
    splits = int(rng.choice([0, 0, 1, 2, 7, 16]))
    keep = float(rng.choice([0.1, 0.5, 1.0]))
    print(f"case: kv4 random chunk heads={G * H}/{H} chunk={L} past={past} keep={keep} splits={splits}", flush=True)
    K, V, kt, vt = _cache(B, H, cap, gpu, seed=seed)
    q = _q(gpu, B, L, G * H, 128, seed=seed)
    lists = _lists(B, H, past, qb, keep, seed=seed)
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past])


@pytest.mark.parametrize("Hq,L", [(32, 1), (16, 16)])
def test_decode_of_131072_tokens(gpu, Hq, L):
    print(f"case: decode4 131072 heads={Hq}/4 q_len={L}", flush=True)
    H, n = 4, 131072
    K, V, kt, vt = _big_cache(H, n // 64, gpu, seed=L)
    q = _q(gpu, 1, L, Hq, 128, seed=1)
    out, lse = ops.attn_decode(q, K, V, [n], SCALE, n // 64, H, with_lse=True)
    _check(out, lse, q, K, V, kt, vt, H, [[list(range(n // 64))] * H], [n - L], [n])


def test_chunk_of_2048_over_32768(gpu):
    print("case: chunk4 2048 over 32768 dense", flush=True)
    H, Hq, L, past = 2, 4, 2048, 512
    cap = past + 32
    K, V, kt, vt = _big_cache(H, cap, gpu, seed=7)
    q = _q(gpu, 1, L, Hq, 128, seed=2)
    lists = [[list(range(cap))] * H]
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, [past], SCALE, cap, H, with_lse=True)
    # every 97th query against 64 bits
    for h in range(H):
        k, v = (ref.read_pages(c.tensor[t[h].long().to(gpu)], of_v).reshape(-1, 128)
                for c, t, of_v in ((K, kt, False), (V, vt, True)))
        kpos = torch.arange(64 * cap, device=gpu)
        for t in range(0, L, 97):
            rows = q[0, t, 2 * h:2 * h + 2].double()
            o, ls, A, S = ref.attention(rows, k, v, kpos, torch.full((2,), 64 * past + t, device=gpu), SCALE)
            assert ((out[0, t, 2 * h:2 * h + 2].double() - o).abs() <= ref.tolerance(o, A, S)).all(), (h, t)
            assert ((lse[0, 2 * h:2 * h + 2, t].double() - ls).abs() <= ref.lse_tolerance(S)).all(), (h, t)


# launches of more than 12 blocks of 256 rows for every CU take the kernel with tiles of 256 rows
LARGE = [
    # (Hq, Hkv, chunk, past blocks, kept share, splits)
    (16, 16, 300, [100], 1.0, 0), (16, 16, 300, [100], 0.4, 1), (8, 8, 161, [200, 230], 0.7, 2), (28, 4, 150, [300, 20, 150], 0.8, 0),
    (24, 6, 400, [130], 1.0, 3), (32, 8, 512, [60, 61], 0.5, 0), (16, 1, 1000, [100], 0.3, 16), (12, 12, 257, [120, 3], 0.05, 4),
]


@pytest.mark.parametrize("Hq,H,L,past,keep,splits", LARGE)
def test_chunks_in_large_tiles(gpu, Hq, H, L, past, keep, splits):
    print(f"case: chunk4 large heads={Hq}/{H} chunk={L} past={past} keep={keep} splits={splits}", flush=True)
    B, qb = len(past), -(-L // 64)
    cap = max(past) + qb
    assert H * -(-L * (Hq // H) // 256) * sum(p + qb for p in past) > 12 * 256 and L * (Hq // H) > 160
    K, V, kt, vt = _big_cache(B * H, cap, gpu, seed=L)
    q = _q(gpu, B, L, Hq, 128, seed=L)
    lists = _lists(B, H, past, qb, keep, seed=L)
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past], every=3)


@pytest.mark.parametrize("splits", [1, 3])
def test_large_tiles_with_odd_lists_and_nan(gpu, splits):
    """Empty lists, unordered ones, and NaN in hidden and in seen places, in tiles of 256 rows."""
    print(f"case: chunk4 large odd lists splits={splits}", flush=True)
    H, Hq, L, past = 16, 16, 300, [100]
    cap = 105
    K, V, kt, vt = _big_cache(H, cap, gpu, seed=1)
    rng = np.random.default_rng(2)
    own = list(range(100, 105))
    lists = [[[] if h == 0 else [104] if h == 1 else own + rng.permutation(100)[:40].tolist() if h == 2 else
              sorted(rng.permutation(100)[:int(rng.integers(1, 100))].tolist()) + own for h in range(H)]]
    lists[0][3] = [7, 7, 9] + own[::-1]
    for h in range(H):  # behind the last token, and in a block that no list names
        for pos in range(6400 + L, 64 * cap):
            _poison(K, V, kt, vt, h, pos, {"k": range(4), "v": range(4)})
        free = min(set(range(100)) - set(lists[0][h]))
        _poison(K, V, kt, vt, h, 64 * free + 3, {"k": range(4), "v": range(4)})
    q = _q(gpu, 1, L, Hq, 128, seed=3)
    table, counts = _tables(lists, cap, gpu)
    args = (q, K, V, table, counts, past, SCALE, cap, H)
    out, lse = ops.attn_fwd(*args, with_lse=True, num_splits=splits)
    assert torch.isfinite(out).all() and (out[0, :, 0] == 0).all() and torch.isneginf(lse[0, 0]).all()
    assert (out[0, :256, 1] == 0).all() and torch.isneginf(lse[0, 1, :256]).all()
    _check(out, lse, q, K, V, kt, vt, H, lists, [6400], [6400 + L])
    _poison(K, V, kt, vt, 2, 6400 + 130, {"v": [2]})
    _poison(K, V, kt, vt, 3, 6400 + 290, {"v": [0], "k": [1]})
    _poison(K, V, kt, vt, 4, 64 * lists[0][4][0] + 9, {"v": [3]})  # seen by all, in a block that is not masked
    out, lse = ops.attn_fwd(*args, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [6400], [6400 + L])
    assert torch.isfinite(out[0, :130, 2]).all() and torch.isnan(out[0, 130:, 2, 64:96]).all()
    assert torch.isfinite(out[0, :290, 3]).all() and torch.isnan(out[0, 290:, 3]).all()
    assert torch.isnan(out[0, :, 4, 96:]).all() and torch.isfinite(out[0, :, 4, :96]).all()


@pytest.mark.parametrize("keep", [1.0, 0.4])
def test_chunks_of_very_unequal_requests(gpu, keep):
    """Split counts of their own for every request (3 or 4 and 1), units dealt by their blocks."""
    B, H, Hq, L, past = 3, 8, 32, 300, [3, 420, 17]
    print(f"case: kv4 chunks of unequal requests keep={keep}", flush=True)
    qb = -(-L // 64)
    cap = max(past) + qb
    K, V, kt, vt = _big_cache(B * H, cap, gpu, seed=21)
    q = _q(gpu, B, L, Hq, 128, seed=22)
    lists = _lists(B, H, past, qb, keep, seed=23)
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past], every=3)


def test_one_long_request_among_many(gpu):
    """480 KV rows whose splits are more than the plan places one by one: whole rows with counts that differ."""
    B, H, Hq, L = 60, 8, 8, 300
    past = [300] + [b % 3 for b in range(1, B)]
    print("case: kv4 one long request among 60", flush=True)
    qb = -(-L // 64)
    cap = max(past) + qb
    K, V, kt, vt = _big_cache(B * H, cap, gpu, seed=31)
    q = _q(gpu, B, L, Hq, 128, seed=32)
    lists = _lists(B, H, past, qb, 0.8, seed=33)
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past], every=7)


def test_drafts_in_large_tiles(gpu):
    """More than 160 packed rows over the whole cache."""
    print("case: decode4 large tiles", flush=True)
    B, H, Hq, L = 2, 4, 64, 64
    lens = [64 * 100 + 5, 64 * 120]
    K, V, kt, vt = _big_cache(B * H, 120, gpu, seed=4)
    assert H * 4 * (101 + 120) > 12 * 256
    q = _q(gpu, B, L, Hq, 128, seed=5)
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    for splits in (0, 1, 5):
        out, lse = ops.attn_decode(q, K, V, lens, SCALE, 120, H, with_lse=True, num_splits=splits)
        _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)


def test_two_streams_at_once(gpu):
    """Calls that overlap on two streams, each with outputs and workspaces of its own, give what they give alone."""
    print("case: kv4 two streams", flush=True)
    H, Hq = 4, 32
    K, V, kt, vt = _big_cache(H, 512, gpu, seed=11)
    qs = [_q(gpu, 1, 1, Hq, 128, seed=s) for s in range(2)]
    qc = _q(gpu, 1, 256, Hq, 128, seed=5)
    table, counts = _tables([[list(range(0, 512, 3)) + [511]] * H], 512, gpu)

    def work(q):
        a = ops.attn_decode(q, K, V, [32768], SCALE, 512, H)
        b = ops.attn_fwd(qc, K, V, table, counts, [508], SCALE, 512, H)
        return a, b

    want = [[t.clone() for t in work(q)] for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[i]))


def test_attention_refuses(gpu):
    K, V, kt, vt = _cache(1, 2, 3, gpu, seed=0)
    q = _q(gpu, 1, 1, 8, 128)
    K16 = ops.KV.heads_first(torch.zeros((1, 2, 192, 128), dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError, match="both"):
        ops.attn_decode(q, K, K16, [100], SCALE, 3, 2)
    with pytest.raises(ValueError, match="cover"):
        ops.attn_decode(q, K, V, [193], SCALE, 4, 2)
    with pytest.raises(ValueError, match="cover"):
        ops.attn_decode(q, K, V, [100], SCALE, 3, 3)
    with pytest.raises(ops._hip.CaError):
        ops.attn_decode(q, K, V, [0], SCALE, 3, 2)
    with pytest.raises(ops._hip.CaError):
        ops.attn_decode(q, K, V, [100], -1.0, 3, 2)
    with pytest.raises(ValueError, match="4352"):
        ops.KV4.paged(K.tensor[:, :4096], K.page_table)
    with pytest.raises(ValueError, match="uint8"):
        ops.KV4.paged(K.tensor.view(torch.int8), K.page_table)
    with pytest.raises(ValueError, match="rows"):
        ops.KV4.paged(K.tensor, K.page_table.t())
    with pytest.raises(ValueError, match="cover"):
        ops.append_q4(q[:, :, :2], q[:, :, :2], K, V, 192, 4)
    with pytest.raises(ops._hip.CaError):
        ops.append_q4(q[:, :, :2], q[:, :, :2], K, V, -1, 3)
    with pytest.raises(ValueError, match="per-request"):
        ops.append_q4(q[:, :, :2], q[:, :, :2], K, V, [1, 2], 3)
    with pytest.raises(ValueError, match="cover"):
        ops.gather_q4(K, V, 1, 2, 100, 93)
    with pytest.raises(ValueError, match="length"):
        ops.gather_q4(K, V, 1, 2, 0, -1)
    none = ops.gather_q4(K, V, 1, 2, 0, 0)
    assert none[0].shape == none[1].shape == (1, 2, 0, 128)
    before = K.tensor.clone()
    ops.append_q4(q[:, :0, :2], q[:, :0, :2], K, V, 0, 3)
    assert torch.equal(K.tensor, before)
