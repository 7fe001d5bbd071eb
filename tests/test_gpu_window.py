"""Attention under a sliding window with sink tokens against its definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from compactattention_amd import ops
from tests.bounded_oracle import BLOCK, D, SCALE, Cache, attention, blocks_seen, random_kv, random_q, visible

pytestmark = pytest.mark.gpu
HUGE = (1 << 31) - 1


def setup(starts, L, Hq, Hkv, W, S, kind, seed=0, mapped=True, **kw):
    N = max(starts) + L
    k, v = random_kv(len(starts), Hkv, N, seed)
    blocks = None
    if mapped and kind in ("paged", "q4"):
        blocks = set()
        for s in starts:
            blocks |= set(blocks_seen(s, L, W, S))
    return Cache(k, v, kind, "cuda", seed, blocks), random_q(len(starts), L, Hq, seed, "cuda", **kw)


def check(out, lse, cache, q, starts, W, S):
    ref, rlse, tol, ltol = attention(q, cache, starts, W, S)
    bad = (out.double().cpu() - ref).abs() > tol
    assert not bad.any(), (bad.nonzero()[:4].tolist(), float(((out.double().cpu() - ref).abs() / tol).max()))
    assert ((lse.double().cpu() - rlse).abs() <= ltol).all()


# (starts, queries, Q heads, KV heads, window, sinks)
CASES = [
    ([0], 1, 4, 1, 1, 0), ([0], 1, 4, 4, 5, 3), ([63], 1, 8, 2, 1, 0), ([64], 1, 8, 2, 64, 0), ([64], 1, 8, 2, 65, 1),
    ([700], 1, 8, 2, 63, 64), ([700], 1, 16, 1, 128, 65), ([1000, 3, 64, 515], 1, 7, 1, 100, 5), ([4000], 1, 4, 2, 1500, 200),
    ([4000], 1, 4, 2, HUGE, 0), ([900], 1, 4, 2, 2, HUGE), ([300], 2, 8, 2, 1, 0), ([300, 0], 4, 8, 2, 70, 4),
    ([510], 5, 8, 2, 66, 63), ([1023], 16, 16, 2, 17, 1), ([129], 16, 7, 1, 300, 130),
    ([0], 64, 4, 1, 1, 0), ([0], 65, 4, 1, 64, 2), ([37], 63, 4, 1, 33, 70), ([640], 64, 2, 2, 128, 64),
    ([1000, 0, 200], 130, 7, 1, 250, 20), ([2048], 129, 8, 1, 640, 4), ([1217], 257, 3, 3, 500, 0), ([100], 200, 4, 1, HUGE, 0),
    ([600], 200, 4, 1, 1, HUGE), ([4096], 70, 16, 1, 1024, 1),
]


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("starts,L,Hq,Hkv,W,S", CASES)
def test_against_definition(starts, L, Hq, Hkv, W, S, kind):
    cache, q = setup(starts, L, Hq, Hkv, W, S, kind, seed=L + W % 97, strided=True)
    out, lse = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, Hkv, with_lse=True)
    check(out, lse, cache, q, starts, W, S)


@pytest.mark.parametrize("kind", ["paged", "q4"])
@pytest.mark.parametrize("L", [1, 6, 90])
@pytest.mark.parametrize("splits", [1, 2, 7, 64])
def test_splits(kind, L, splits):
    starts, W, S = [1500, 333], 900, 70
    cache, q = setup(starts, L, 8, 2, W, S, kind, seed=splits)
    out, lse = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, 2, with_lse=True, num_splits=splits)
    check(out, lse, cache, q, starts, W, S)


# chunks that run in tiles of 128 rows, where two waves share rows and take blocks in turn, and in tiles of 256
CHUNKS = [([900, 64], 600, 16, 2, 400, 3), ([0], 1300, 8, 1, 900, 0), ([500], 2000, 7, 7, 100, 3), ([300], 2100, 16, 8, 200, 3)]


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("starts,L,Hq,Hkv,W,S", CHUNKS)
def test_chunks(starts, L, Hq, Hkv, W, S, kind):
    cache, q = setup(starts, L, Hq, Hkv, W, S, kind, seed=L, strided=True)
    out, lse = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, Hkv, with_lse=True)
    check(out, lse, cache, q, starts, W, S)


@pytest.mark.parametrize("case,splits,kind", [(0, 2, "paged"), (0, 3, "paged"), (0, 64, "paged"), (1, 5, "paged"), (3, 3, "paged"), (0, 5, "q4"),
                                              (3, 3, "q4")])
def test_splits_of_chunks(case, splits, kind):
    starts, L, Hq, Hkv, W, S = CHUNKS[case]
    cache, q = setup(starts, L, Hq, Hkv, W, S, kind, seed=splits)
    out, lse = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, Hkv, with_lse=True, num_splits=splits)
    check(out, lse, cache, q, starts, W, S)


@pytest.mark.parametrize("case,splits,kind", [(0, 0, "paged"), (0, 2, "paged"), (3, 0, "paged"), (3, 2, "paged"), (0, 0, "q4"), (3, 0, "q4")])
def test_chunks_with_values_that_are_not_finite(case, splits, kind):
    """Hidden from all queries: no effect.  Visible: a value in its dims (in 4 bits NaN in its group's), a NaN key in the whole
    output and the lse."""
    starts, L, Hq, Hkv, W, S = CHUNKS[case]
    k, v = random_kv(len(starts), Hkv, max(starts) + L, 8)
    for b, start in enumerate(starts):
        for i, bad in enumerate((math.nan, math.inf, -math.inf)):
            hidden = slice(S + i, max(S + i, start - W + 1), 3)
            k[b, :, hidden], v[b, :, hidden] = bad, bad
        for i, j in enumerate((1, start + 5, start + L // 3, start + L - 70, start + L - 1)):
            v[b, i % Hkv, j, 17 * i] = (math.inf, -math.inf, math.nan)[i % 3]
    k[-1, 0, starts[-1] + L // 2, 9] = math.nan
    cache, q = Cache(k, v, kind, "cuda", 8), random_q(len(starts), L, Hq, 8, "cuda")
    out, lse = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, Hkv, with_lse=True, num_splits=splits)
    out, lse = out.cpu().double(), lse.cpu().double()
    ref, rlse, _, ltol = attention(q, cache, starts, W, S)
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(torch.isnan(lse), torch.isnan(rlse))
    assert torch.isnan(rlse).any() and torch.isfinite(rlse).any() and (kind == "q4" or torch.isinf(ref).any())
    there = torch.isfinite(rlse)
    assert ((lse - rlse).abs()[there] <= ltol[there]).all()
    fin = torch.isfinite(ref)
    infinite = torch.isinf(ref)
    assert torch.equal(out[infinite], ref[infinite])
    cache.v = torch.where(torch.isfinite(cache.v), cache.v, 0.0)  # the tolerance of what is finite
    _, _, tol, _ = attention(q, cache, starts, W, S)
    assert ((out - ref).abs()[fin] <= tol[fin]).all()


def test_long_chunk_of_many_tiles():
    # several row tiles a row, most of the loop unmasked, one start for all, the sequence-first layout and out given
    starts, L, W, S = [2000, 2000], 300, 1300, 66
    cache, q = setup(starts, L, 8, 2, W, S, "seq", seed=5)
    out = torch.empty_like(q)
    got, lse = ops.attn_window(q, cache.K, cache.V, 2000, W, S, SCALE, cache.cap, 2, out=out, with_lse=True)
    assert got is out
    check(out, lse, cache, q, starts, W, S)


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("L,W,S,start", [(1, 100, 5, 777), (3, 100, 70, 777), (9, 40, 3, 500), (100, 70, 66, 400), (300, 150, 1, 333)])
def test_what_every_query_hides_has_no_effect(kind, L, W, S, start):
    """NaN and infinities in all keys and values that no query sees, those of the blocks with visible keys among them."""
    Hq, Hkv = 8, 2
    cache, q = setup([start], L, Hq, Hkv, W, S, kind, mapped=False)
    kpos = torch.arange(cache.N)
    seen = torch.zeros(cache.N, dtype=torch.bool)
    for t in range(L):
        seen |= visible(start + t, kpos, W, S)
    want, wlse = ops.attn_window(q, cache.K, cache.V, [start], W, S, SCALE, cache.cap, Hkv, with_lse=True)
    k, v = random_kv(1, Hkv, cache.N, 0)
    for i, bad in enumerate((math.nan, math.inf, -math.inf)):
        hidden = (~seen).nonzero()[i::3, 0]
        k[:, :, hidden], v[:, :, hidden] = bad, bad
    poisoned = Cache(k, v, kind, "cuda", 0)
    got, glse = ops.attn_window(q, poisoned.K, poisoned.V, [start], W, S, SCALE, cache.cap, Hkv, with_lse=True)
    assert torch.equal(glse, wlse)
    # (keys of a block with such a value are taken one by one, another order of the same sums)
    check(got, glse, cache, q, [start], W, S)
    if kind == "q4":
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["paged", "q4"])
@pytest.mark.parametrize("L,W,S", [(1, 100, 5), (4, 64, 3), (10, 40, 70), (90, 50, 3), (280, 100, 0)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_the_queries_that_see_them(kind, L, W, S, bad):
    start, Hq, Hkv = 450, 8, 2
    N = start + L
    k, v = random_kv(1, Hkv, N, 3)
    at = sorted({1, S + 1, start - W, start - W // 2, start - 1, start, start + L // 2, N - 1, start + max(0, L - W - 3)})
    at = [j for j in at if 0 <= j < N]
    for i, j in enumerate(at):
        v[0, i % Hkv, j, (17 * i) % D] = bad
    cache, q = Cache(k, v, kind, "cuda", 3), random_q(1, L, Hq, 3, "cuda")
    out = ops.attn_window(q, cache.K, cache.V, [start], W, S, SCALE, cache.cap, Hkv).cpu().double()
    ref, _, _, _ = attention(q, cache, [start], W, S)
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    fin = torch.isfinite(ref)
    infinite = ~fin & ~torch.isnan(ref)
    assert torch.equal(out[infinite], ref[infinite])
    cache.v = torch.where(torch.isfinite(cache.v), cache.v, 0.0)  # the tolerance of what is finite
    _, _, tol, _ = attention(q, cache, [start], W, S)
    assert ((out - ref).abs()[fin] <= tol[fin]).all()


@pytest.mark.parametrize("kind", ["paged", "q4"])
@pytest.mark.parametrize("L,back", [(1, 30), (5, 30), (100, 30), (5, 58), (70, 0)])
def test_nan_key(kind, L, back):
    start, W, S, Hq, Hkv = 300, 60, 3, 4, 1
    k, v = random_kv(1, Hkv, start + L, 4)
    at = start + L // 2 - back
    k[0, 0, at, 5] = math.nan
    cache, q = Cache(k, v, kind, "cuda", 4), random_q(1, L, Hq, 4, "cuda")
    out, lse = ops.attn_window(q, cache.K, cache.V, [start], W, S, SCALE, cache.cap, Hkv, with_lse=True)
    sees = torch.tensor([bool(visible(start + t, torch.tensor([at]), W, S)) for t in range(L)])
    assert torch.equal(torch.isnan(out.cpu()).all(-1).all(-1)[0], sees) and torch.equal(torch.isnan(out.cpu()).any(-1).any(-1)[0], sees)
    assert torch.equal(torch.isnan(lse.cpu()).all(1)[0], sees)
    assert sees.any() and (L < 70 and back == 30 or not sees.all())  # (of 5 queries all see the key 30 back)


def test_captured_and_on_another_stream():
    starts, L, W, S = [1400, 90], 3, 700, 5
    for kind in ("paged", "q4"):
        cache, q = setup(starts, L, 8, 2, W, S, kind)
        want = ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, 2, num_splits=4)
        out = torch.zeros_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, 2, out=out, num_splits=4)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attn_window(q, cache.K, cache.V, starts, W, S, SCALE, cache.cap, 2, out=out, num_splits=4)
        for i in range(4):
            out.zero_()
            q2 = random_q(2, L, 8, 100 + i, "cuda")
            q.copy_(q2)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.attn_window(q2, cache.K, cache.V, starts, W, S, SCALE, cache.cap, 2, num_splits=4))


@pytest.mark.parametrize("L", [1, 40])
def test_pages_past_4_gib(L):
    """Pages whose bytes lie past 2^32: only those that are read are written before."""
    start, W, S, Hkv = 200, 100, 3, 2
    cache, q = setup([start], L, 4, Hkv, W, S, "paged", seed=9, mapped=False)
    want = ops.attn_window(q, cache.K, cache.V, [start], W, S, SCALE, cache.cap, Hkv)
    pages = (1 << 32) // (BLOCK * D * 2) + 64
    table = (cache.table + (pages - cache.stores[0].shape[0])).contiguous()
    pools = []
    for p in cache.stores:
        pool = torch.empty((pages, BLOCK, D), dtype=torch.bfloat16, device="cuda")
        pool[pages - p.shape[0]:] = p
        pools.append(pool)
    got = ops.attn_window(q, ops.KV.paged(pools[0], table), ops.KV.paged(pools[1], table), [start], W, S, SCALE, cache.cap, Hkv)
    assert torch.equal(got, want)


def test_windows_and_positions_past_32_bits():
    """A window or sinks past 2^31 are as good as everything; nothing is taken modulo 2^32."""
    cache, q = setup([300], 2, 8, 2, HUGE, 0, "paged")
    want = ops.attn_window(q, cache.K, cache.V, [300], 10 ** 6, 0, SCALE, cache.cap, 2)
    for W, S in ((1 << 31, 0), ((1 << 32) + 5, 0), (1, (1 << 32) + 1), (10 ** 12, 10 ** 12)):
        assert torch.equal(ops.attn_window(q, cache.K, cache.V, [300], W, S, SCALE, cache.cap, 2), want)
    for kw in (dict(window=-(1 << 32) + 5), dict(window=0), dict(sinks=-(1 << 32))):
        with pytest.raises(ops._hip.CaError):
            ops.attn_window(q, cache.K, cache.V, [300], **{"window": 5, "sinks": 0, **kw}, scale=SCALE, kv_cap=cache.cap, num_kv_heads=2)
    for bad in (dict(start=[(1 << 32) + 300]), dict(num_splits=1 << 32)):
        with pytest.raises(ValueError):
            ops.attn_window(q, cache.K, cache.V, **{"start": [300], **bad}, window=5, sinks=0, scale=SCALE, kv_cap=cache.cap, num_kv_heads=2)


def test_what_the_entry_point_refuses():
    cache, q = setup([100], 3, 8, 2, 50, 0, "paged")
    q4, _ = setup([100], 3, 8, 2, 50, 0, "q4")
    args = (50, 0, SCALE, cache.cap, 2)
    with pytest.raises(ValueError, match="all be bf16 or all be held"):
        ops.attn_window(q, cache.K, q4.V, [100], *args)
    with pytest.raises(ValueError, match="does not cover"):
        ops.attn_window(q, cache.K, cache.V, [200], *args)
    with pytest.raises(ValueError, match="per-request"):
        ops.attn_window(q, cache.K, cache.V, [100, 100], *args)
    with pytest.raises(ValueError, match="q's shape"):
        ops.attn_window(q, cache.K, cache.V, [100], *args, out=q[:, :2])
    with pytest.raises(ValueError, match="bfloat16"):
        ops.attn_window(q.float(), cache.K, cache.V, [100], *args)
    empty, lse = ops.attn_window(q[:, :0], cache.K, cache.V, [100], *args, with_lse=True)
    assert empty.shape == (1, 0, 8, 128) and lse.shape == (1, 8, 0)


def test_two_calls_at_once():
    """Calls on two streams have workspaces of their own."""
    a, qa = setup([3000], 40, 8, 2, 2000, 5, "paged", seed=1)
    b, qb = setup([2500], 40, 8, 2, 1500, 5, "paged", seed=2)
    run = [lambda o=None: ops.attn_window(qa, a.K, a.V, [3000], 2000, 5, SCALE, a.cap, 2, num_splits=8, out=o),
           lambda o=None: ops.attn_window(qb, b.K, b.V, [2500], 1500, 5, SCALE, b.cap, 2, num_splits=8, out=o)]
    want = [f() for f in run]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
