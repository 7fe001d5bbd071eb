"""Eviction by accumulated weight: which tokens stay, and their move, exactly."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from compactattention_amd import ops
from tests import kv4_oracle
from tests.bounded_oracle import Cache, kept, random_kv

pytestmark = pytest.mark.gpu


def want_keep(mass, lens, Hkv, budget, sinks, recent):
    m = mass.cpu().numpy()
    out = np.full((m.shape[0], budget), -1, np.int32)
    for r in range(m.shape[0]):
        ids = kept(m[r], lens[r // Hkv], budget, sinks, recent)
        out[r, :len(ids)] = ids
    return torch.from_numpy(out)


def masses(rows, n, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.exp(3 * torch.randn((rows, n), generator=g))
    if kind == "ties":
        x = torch.randint(0, 4, (rows, n), generator=g).float()
    elif kind == "equal":
        x = torch.full((rows, n), 0.25)
    elif kind == "close":  # agree in all but the last bits
        x = (torch.full((rows, n), 1.0).view(torch.int32) + torch.randint(0, 40, (rows, n), generator=g, dtype=torch.int32)).view(torch.float32)
    elif kind == "odd":  # NaN, infinities, signs, zeros of both signs, subnormals
        x = torch.randn((rows, n), generator=g)
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-40, -1e-40, -math.nan])
        pick = torch.randint(0, 24, (rows, n), generator=g)
        x = torch.where(pick < 8, special[pick.clamp(max=7)], x)
    return x.cuda()


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("lens,Hkv,budget,sinks,recent", [
    ([2], 1, 1, 0, 0), ([2], 1, 1, 0, 1), ([2], 1, 1, 1, 0), ([65], 2, 64, 0, 0), ([65], 2, 64, 4, 60), ([130], 1, 64, 64, 0),
    ([1000, 63, 0, 64, 1], 2, 64, 4, 16), ([777], 3, 500, 5, 101), ([5000, 4097], 2, 1000, 4, 500), ([1500], 1, 1499, 3, 7),
    ([40001], 1, 4096, 4, 1024), ([20000], 2, 7, 0, 0),
])
def test_heavy_tokens(kind, lens, Hkv, budget, sinks, recent):
    mass = masses(len(lens) * Hkv, max(lens) + 5, kind, seed=budget)
    keep = ops.heavy_tokens(mass, lens, Hkv, budget, sinks, recent)
    assert torch.equal(keep.cpu(), want_keep(mass, lens, Hkv, budget, sinks, recent))


@pytest.mark.parametrize("share", [0.0, 0.05, 0.2, 0.9])  # of the blocks of 64 keys that any query gave weight
@pytest.mark.parametrize("n", [70, 3000, 16384, 20000, 70000])
def test_weights_of_zero(n, share):
    g = torch.Generator().manual_seed(n)
    some = (torch.rand((2, n // 64 + 1), generator=g) < share).repeat_interleave(64, 1)[:, :n]
    mass = (masses(2, n, "spread", n).cpu() * some * torch.randint(-1, 2, (2, n), generator=g).abs()).cuda()
    for budget in (n // 10, n // 2, n - 5):
        keep = ops.heavy_tokens(mass, n, 2, budget, 3, 4)
        assert torch.equal(keep.cpu(), want_keep(mass, [n], 2, budget, 3, 4)), budget


@pytest.mark.parametrize("columns", [0, 5])
def test_requests_without_tokens(columns):
    mass = torch.ones((4, columns), device="cuda")
    keep = ops.heavy_tokens(mass, [0, 0], 2, 70, 2, 3)
    assert torch.equal(keep.cpu(), torch.full((4, 70), -1, dtype=torch.int32))
    pool = torch.ones((8, 64, 128), dtype=torch.bfloat16, device="cuda")
    K = ops.KV.paged(pool, torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2))
    moved = ops.move_tokens(K, K, K, K, keep, [0, 0], 2, mass=mass)
    assert torch.equal(moved.cpu(), torch.zeros((4, 70))) and bool((pool == 1).all())


def test_strided_mass_and_many_rows():
    mass = masses(64 * 8, 300, "ties", 1)
    lens = [37 + 4 * b for b in range(64)]
    keep = ops.heavy_tokens(mass[:, :290], lens, 8, 50, 2, 10)
    assert torch.equal(keep.cpu(), want_keep(mass, lens, 8, 50, 2, 10))


def test_long_rows():
    mass = masses(2, 200000, "spread", 2)
    keep = ops.heavy_tokens(mass, 200000, 2, 8191, 4, 1023)
    assert torch.equal(keep.cpu(), want_keep(mass, [200000], 2, 8191, 4, 1023))


def dest(kind, B, H, n, seed):
    """An empty destination (bytes of 0x5a), its store tensors and layouts."""
    blocks = -(-n // 64)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * H * blocks, generator=g).to(torch.int32).view(B * H, blocks).cuda()
    out = []
    for _ in range(2):
        if kind == "q4":
            t = torch.full((B * H * blocks, kv4_oracle.PAGE), 0x5a, dtype=torch.uint8, device="cuda")
            out.append((t, ops.KV4.paged(t, table)))
        elif kind == "paged":
            t = torch.full((B * H * blocks, 64, 128), 7.0, dtype=torch.bfloat16, device="cuda")
            out.append((t, ops.KV.paged(t, table)))
        else:
            t = torch.full((B, H, n, 128), 7.0, dtype=torch.bfloat16, device="cuda")
            out.append((t, ops.KV.heads_first(t)))
    return out, table


def token_bytes(t, of_v):
    code = sorted({kv4_oracle.code_at(t, d, of_v) for d in range(128)})
    return code + [kv4_oracle.scale_at(t, g, of_v) for g in range(4)]


@pytest.mark.parametrize("kind", ["paged", "heads", "q4"])
@pytest.mark.parametrize("lens,H,n", [([1], 1, 1), ([100], 2, 64), ([300, 40, 0], 2, 65), ([1000, 130], 1, 333), ([64], 1, 100)])
def test_move_tokens(kind, lens, H, n):
    B = len(lens)
    k, v = random_kv(B, H, max(lens), 4)
    cache = Cache(k, v, kind, "cuda", 4)
    mass = masses(B * H, max(lens), "spread", 5)
    keep = ops.heavy_tokens(mass, lens, H, n, 0, min(3, n))
    (kd, K2), (vd, V2) = dest(kind, B, H, n, 6)[0]
    before = [kd.clone(), vd.clone()]
    moved = ops.move_tokens(cache.K, cache.V, K2, V2, keep, lens, H, mass=mass)
    ids = keep.cpu()
    for b in range(B):
        c = min(n, lens[b])
        for h in range(H):
            r = b * H + h
            at = ids[r, :c].long()
            assert torch.equal(moved[r, :c].cpu(), mass[r].cpu()[at]) and (moved[r, c:] == 0).all()
            for store, src, x, of_v, was in ((kd, cache.stores[0], k, False, before[0]), (vd, cache.stores[1], v, True, before[1])):
                if kind == "heads":
                    assert torch.equal(store[b, h, :c].cpu(), x[b, h, at])
                    assert torch.equal(store[b, h, c:], was[b, h, c:])
                    continue
                layout = K2 if not of_v else V2
                table, stable = layout.page_table[r].cpu(), cache.table[r].cpu()
                got, orig, old = store.cpu(), src.cpu(), was.cpu()
                expect = old[table.long()].clone()
                for i, j in enumerate(at.tolist()):
                    if kind == "paged":
                        expect[i // 64, i % 64] = orig[stable[j // 64], j % 64]
                    else:
                        expect[i // 64, token_bytes(i % 64, of_v)] = orig[stable[j // 64], token_bytes(j % 64, of_v)]
                assert torch.equal(got[table.long()], expect)


def test_move_inside_one_pool_and_bad_ids():
    """Source and destination pages of one pool; destination ids outside the pool are passed over, positions outside a row
    are taken into it."""
    k, v = random_kv(1, 1, 256, 8)
    cache = Cache(k, v, "paged", "cuda", 8)
    pools = [torch.cat([p, torch.zeros((3, 64, 128), dtype=p.dtype, device="cuda")]) for p in cache.stores]
    first = cache.stores[0].shape[0]
    table = torch.tensor([[first + 1, -1, first + 7]], dtype=torch.int32, device="cuda")  # one page, two ids outside
    keep = torch.arange(10, 202, dtype=torch.int32, device="cuda")[None].contiguous()
    keep[0, 5], keep[0, 6] = -7, 1 << 30
    src = [ops.KV.paged(p, cache.table) for p in pools]
    dst = [ops.KV.paged(p, table) for p in pools]
    before = [p.clone() for p in pools]
    ops.move_tokens(*src, *dst, keep, 256, 1)
    torch.cuda.synchronize()
    for p, was, x in zip(pools, before, (k, v)):
        want = x[0, 0, 10:74].clone()
        want[5], want[6] = x[0, 0, 0], x[0, 0, 255]
        assert torch.equal(p[first + 1].cpu(), want)
        was[first + 1] = p[first + 1]
        assert torch.equal(p.view(torch.int16), was.view(torch.int16))


def test_captured():
    mass = masses(4, 3000, "spread", 9)
    keep = torch.empty((4, 100), dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = ops.heavy_tokens(mass, 3000, 4, 100, 4, 10)
    for i in range(4):
        mass.copy_(masses(4, 3000, "ties" if i % 2 else "spread", 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keep.cpu(), want_keep(mass, [3000], 4, 100, 4, 10))
        assert torch.equal(keep, ops.heavy_tokens(mass, 3000, 4, 100, 4, 10))


def test_what_the_entry_points_refuse():
    mass = masses(4, 300, "spread", 30)
    with pytest.raises(ValueError, match="KV heads"):
        ops.heavy_tokens(mass, 300, 3, 10)
    with pytest.raises(ValueError, match="mass"):
        ops.heavy_tokens(mass, 301, 4, 10)
    with pytest.raises(ValueError, match="32 bits"):
        ops.heavy_tokens(mass, 300, 4, (1 << 32) + 10)
    for bad in (dict(budget=0), dict(budget=10, sinks=-1), dict(budget=10, sinks=6, recent=5)):
        with pytest.raises(ops._hip.CaError):
            ops.heavy_tokens(mass, 300, 4, **bad)
    k, v = random_kv(1, 4, 300, 31)
    cache = Cache(k, v, "paged", "cuda", 31)
    q4 = Cache(k, v, "q4", "cuda", 31)
    keep = ops.heavy_tokens(mass, 300, 4, 100)
    (_, K2), (_, V2) = dest("paged", 1, 4, 100, 32)[0]
    (_, K64), _ = dest("paged", 1, 4, 64, 32)[0]
    with pytest.raises(ValueError, match="all be bf16 or all be held"):
        ops.move_tokens(q4.K, q4.V, K2, V2, keep, 300, 4)
    with pytest.raises(ValueError, match="k_dst"):
        ops.move_tokens(cache.K, cache.V, K64, V2, keep, 300, 4)
    with pytest.raises(ValueError, match="does not cover"):
        ops.move_tokens(cache.K, cache.V, K2, V2, keep, 400, 4)
    with pytest.raises(ValueError, match="int32"):
        ops.move_tokens(cache.K, cache.V, K2, V2, keep.long(), 300, 4)
    assert ops.move_tokens(cache.K, cache.V, K2, V2, keep, 300, 4) is None


def test_two_calls_at_once():
    a, b = masses(8, 50000, "spread", 40), masses(8, 40000, "ties", 41)
    want = [ops.heavy_tokens(a, 50000, 8, 3000, 4, 100), ops.heavy_tokens(b, 40000, 8, 2000, 0, 50)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        with torch.cuda.stream(streams[0]):
            got[0].append(ops.heavy_tokens(a, 50000, 8, 3000, 4, 100))
        with torch.cuda.stream(streams[1]):
            got[1].append(ops.heavy_tokens(b, 40000, 8, 2000, 0, 50))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_long_rows_captured():
    """The launches of rows in slices, replayed with other weights in place."""
    mass = masses(4, 40000, "spread", 50)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = ops.heavy_tokens(mass, [40000, 17000], 2, 1000, 4, 10)
    for i in range(4):
        mass.copy_(masses(4, 40000, ("ties", "spread", "close", "odd")[i], 60 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keep.cpu(), want_keep(mass, [40000, 17000], 2, 1000, 4, 10))
        assert torch.equal(keep, ops.heavy_tokens(mass, [40000, 17000], 2, 1000, 4, 10))
