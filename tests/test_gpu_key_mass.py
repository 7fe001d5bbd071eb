"""The attention weight that keys receive against its definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from compactattention_amd import ops
from tests.bounded_oracle import SCALE, Cache, attention, random_kv, random_q, weights

pytestmark = pytest.mark.gpu


def setup(starts, L, Hq, Hkv, kind, seed, window=0, sinks=0):
    k, v = random_kv(len(starts), Hkv, max(starts) + L, seed)
    cache, q = Cache(k, v, kind, "cuda", seed), random_q(len(starts), L, Hq, seed, "cuda", strided=True)
    _, lse, _, _ = attention(q, cache, starts, window or 1 << 30, sinks)
    g = torch.Generator().manual_seed(seed)
    mass = torch.rand((len(starts) * Hkv, cache.cap * 64), generator=g).cuda()
    return cache, q, lse.float().cuda(), mass


def check(got, mass, q, cache, lse, starts, window=0, sinks=0, lists=None):
    ref, tol = weights(q, cache, lse, mass, starts, window, sinks, lists)
    L = q.shape[1]
    for b, s in enumerate(starts):
        rows = slice(b * cache.H, (b + 1) * cache.H)
        diff = (got.cpu().double() - ref).abs()[rows, :s + L]
        assert (diff <= tol[rows, :s + L]).all(), float((diff / tol[rows, :s + L]).max())
        # behind the last token nothing is written
        assert torch.equal(got[rows, s + L:], mass[rows, s + L:].to(got.device))


CASES = [([0], 1, 4, 1), ([63], 1, 4, 4), ([64], 1, 8, 2), ([1000, 3, 64, 515], 1, 7, 1), ([700], 2, 16, 1), ([129, 0], 16, 7, 1),
         ([37], 63, 4, 1), ([0], 65, 4, 1), ([500, 130], 130, 8, 2), ([300], 257, 3, 3), ([0], 300, 16, 1)]


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("starts,L,Hq,Hkv", CASES)
def test_against_definition(starts, L, Hq, Hkv, kind):
    cache, q, lse, mass = setup(starts, L, Hq, Hkv, kind, seed=L)
    old = mass.clone()
    got = ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cache.cap, Hkv)
    assert got is mass
    check(got, old, q, cache, lse, starts)
    out = old.clone()
    out[:, :] = old
    again = ops.key_mass(q, cache.K, lse, old, starts, SCALE, cache.cap, Hkv, out=out)
    assert again is out and torch.equal(out, mass)  # the same order of sums


@pytest.mark.parametrize("kind", ["paged", "q4"])
@pytest.mark.parametrize("starts,L,W,S", [([300], 1, 1, 0), ([300], 1, 64, 5), ([700, 20], 5, 100, 70), ([200], 150, 33, 1),
                                          ([640], 200, 128, 64), ([100], 90, 1 << 31 - 1, 0), ([500], 100, 3, 2000)])
def test_window(kind, starts, L, W, S):
    W = min(W, (1 << 31) - 1)
    cache, q, lse, mass = setup(starts, L, 8, 2, kind, seed=L + 1, window=W, sinks=S)
    old = mass.clone()
    ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cache.cap, 2, window=W, sinks=S)
    check(mass, old, q, cache, lse, starts, W, S)


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("starts,L", [([640], 1), ([1280, 70], 3), ([700], 200), ([0, 1984, 130], 64)])
def test_lists(kind, starts, L):
    Hkv = 2
    cache, q, lse, mass = setup(starts, L, 8, Hkv, kind, seed=L + 2)
    rows, cap = len(starts) * Hkv, cache.cap + 3
    g = torch.Generator().manual_seed(L)
    table, counts, lists = torch.full((rows, cap), -1, dtype=torch.int32), [], []
    for r in range(rows):
        nkb = -(-(starts[r // Hkv] + L) // 64)
        keep = (torch.rand(nkb, generator=g) < 0.5).nonzero()[:, 0].tolist()
        if r == 1:
            keep = []  # a list without blocks
        if r == 2:
            keep = list(range(nkb))
        lists.append(keep)
        counts.append(len(keep))
        table[r, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    table, counts = table.cuda(), torch.tensor(counts, dtype=torch.int32).cuda()
    old = mass.clone()
    out = old.clone()
    ops.key_mass(q, cache.K, lse, old, starts, SCALE, cap, Hkv, table=table, counts=counts, out=out)
    check(out, old, q, cache, lse, starts, lists=lists)
    # what no list names is copied (a key's place that held something else before)
    out2 = torch.full_like(old, 7.0)
    ops.key_mass(q, cache.K, lse, old, starts, SCALE, cap, Hkv, table=table, counts=counts, out=out2)
    for b, s in enumerate(starts):
        sl = slice(b * Hkv, (b + 1) * Hkv)
        assert torch.equal(out2[sl, :s + L], out[sl, :s + L]) and (out2[sl, s + L:] == 7.0).all()
    ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cap, Hkv, table=table, counts=counts)
    assert torch.equal(mass, out)


def test_last_tokens_of_a_chunk():
    """q and lse as slices of a chunk's: the weights of its last tokens alone."""
    cache, q, lse, mass = setup([300], 100, 8, 2, "paged", seed=11)
    old = mass.clone()
    ops.key_mass(q[:, -33:], cache.K, lse[:, :, -33:], mass, [367], SCALE, cache.cap, 2)
    check(mass, old, q[:, -33:], cache, lse[:, :, -33:], [367])


@pytest.mark.parametrize("L", [1, 70])
def test_queries_without_a_key_and_nan(L):
    cache, q, lse, mass = setup([150], L, 8, 2, "paged", seed=12)
    old = mass.clone()
    lse[0, 1, L // 2] = -math.inf  # adds nothing
    lse[0, 3, L - 1] = math.inf    # likewise: exp(-inf)
    ops.key_mass(q, cache.K, lse, mass, [150], SCALE, cache.cap, 2)
    assert torch.isfinite(mass).all()
    ref = lse.clone()
    ref[0, 3, L - 1] = -math.inf
    check(mass, old, q, cache, ref, [150])
    # a NaN lse: the keys that its query sees, of its KV head
    lse[0, 5, 0] = math.nan
    mass = old.clone()
    ops.key_mass(q, cache.K, lse, mass, [150], SCALE, cache.cap, 2)
    nan = torch.isnan(mass.cpu())
    assert not nan[0].any() and nan[1, :151].all() and not nan[1, 151:].any()


@pytest.mark.parametrize("kind", ["paged", "q4"])
@pytest.mark.parametrize("L", [1, 64, 100])
def test_keys_that_are_not_finite(kind, L):
    start = 200
    k, v = random_kv(1, 1, start + L, 13)
    at = start + L // 2  # hidden from the queries before it
    k[0, 0, at, 3] = math.nan
    q = random_q(1, L, 4, 13, "cuda")
    cache = Cache(k, v, kind, "cuda", 13)
    lse = torch.zeros((1, 4, L), device="cuda") + 5.0
    mass = torch.zeros((1, cache.cap * 64), device="cuda")
    ops.key_mass(q, cache.K, lse, mass, [start], SCALE, cache.cap, 1)
    assert torch.isnan(mass[0, at]) and torch.isfinite(mass).sum() == mass.numel() - 1
    # seen by no query: its weight stays
    mass = torch.zeros((1, cache.cap * 64), device="cuda")
    ops.key_mass(q[:, :1], cache.K, lse[:, :, :1], mass, [at - 2], SCALE, cache.cap, 1)
    assert torch.isfinite(mass).all()


def test_captured_and_deterministic():
    starts = [1000, 200]
    cache, q, lse, mass = setup(starts, 40, 8, 2, "paged", seed=14)
    want = ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cache.cap, 2, out=mass.clone())
    out = torch.zeros_like(mass)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cache.cap, 2, out=out)
    for i in range(4):
        out.copy_(mass)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        mass2 = ops.key_mass(q, cache.K, lse, mass, starts, SCALE, cache.cap, 2, out=mass.clone())
        assert torch.equal(mass2, want)


def test_weights_of_a_query_add_up_to_its_heads():
    """With the lse of the same attention the weights of a step sum to the number of query heads of every KV head."""
    cache, q, _, mass = setup([2999], 1, 8, 2, "paged", seed=15)
    mass.zero_()
    _, lse = ops.attn_decode(q, cache.K, cache.V, [3000], SCALE, cache.cap, 2, with_lse=True)
    ops.key_mass(q, cache.K, lse, mass, 2999, SCALE, cache.cap, 2)
    # the lse is that of weights rounded to bf16, off by 2^-8 each at most
    assert ((mass.double().sum(1) - 4).abs() <= 4 * 1.1 * 2.0 ** -8).all()


def test_what_the_entry_point_refuses():
    cache, q, lse, mass = setup([100], 3, 8, 2, "paged", seed=16)
    args = ([100], SCALE, cache.cap, 2)
    for bad, text in ((dict(lse=lse[:, :4]), "lse"), (dict(lse=lse.double()), "float32"), (dict(mass=mass[:1]), "mass"),
                      (dict(mass=mass[:, :102]), "mass"), (dict(mass=mass.half()), "float32"), (dict(mass=mass[:1].expand(2, -1)), "overlap")):
        a = dict(q=q, k=cache.K, lse=lse, mass=mass)
        a.update(bad)
        with pytest.raises(ValueError, match=text):
            ops.key_mass(a["q"], a["k"], a["lse"], a["mass"], *args)
    table = torch.zeros((2, cache.cap), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="both"):
        ops.key_mass(q, cache.K, lse, mass, *args, table=table)
    with pytest.raises(ops._hip.CaError, match="overlap"):
        ops.key_mass(q, cache.K, lse, mass[:, :110], *args, out=mass[:, 5:115])
    with pytest.raises(ops._hip.CaError, match="window"):
        ops.key_mass(q, cache.K, lse, mass, *args, window=-1)
    old = mass.clone()
    assert ops.key_mass(q[:, :0], cache.K, lse[:, :, :0], mass, *args) is mass and torch.equal(mass, old)
    out = torch.zeros_like(mass)
    ops.key_mass(q[:, :0], cache.K, lse[:, :, :0], mass, *args, out=out)
    assert torch.equal(out[:, :100], mass[:, :100]) and (out[:, 100:] == 0).all()


def test_parts_of_a_long_chunk():
    """Enough query tiles over few blocks that parts of them have workgroups of their own, with lists and without."""
    for kind in ("paged", "q4"):
        cache, q, lse, mass = setup([130], 600, 16, 2, kind, seed=17)
        old = mass.clone()
        ops.key_mass(q, cache.K, lse, mass, [130], SCALE, cache.cap, 2)
        check(mass, old, q, cache, lse, [130])
        table = torch.full((2, cache.cap), -1, dtype=torch.int32)
        lists = [[0, 2, 5, 11], list(range(1, 12))]
        for r, x in enumerate(lists):
            table[r, :len(x)] = torch.tensor(x, dtype=torch.int32)
        counts = torch.tensor([4, 11], dtype=torch.int32).cuda()
        out = torch.zeros_like(old)
        out[:, 730:] = old[:, 730:]
        ops.key_mass(q, cache.K, lse, old, [130], SCALE, cache.cap, 2, window=400, sinks=3, table=table.cuda(), counts=counts, out=out)
        check(out, old, q, cache, lse, [130], 400, 3, lists)


def test_the_largest_groups_and_odd_ones():
    for Hq, Hkv in ((11, 1), (13, 1), (30, 2), (16, 1), (5, 5)):
        cache, q, lse, mass = setup([70, 200], 37, Hq, Hkv, "heads", seed=Hq)
        old = mass.clone()
        ops.key_mass(q, cache.K, lse, mass, [70, 200], SCALE, cache.cap, Hkv)
        check(mass, old, q, cache, lse, [70, 200])
