"""Calls on caches of bounded size one after the other, on a cache in host memory whose operators are plain indexing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from compactattention_amd import ops
from compactattention_amd.kv_cache import PagedKVCache
from tests.bounded_oracle import kept


class Plain:
    """A cache's layout as the operators below take it."""

    def __init__(self, pool, page_table):
        self.pool, self.page_table = pool, page_table


def plain_heavy_tokens(mass, n, num_kv_heads, budget, sinks=0, recent=0):
    rows = [kept(m, n, budget, sinks, recent) for m in mass.numpy()]
    return torch.tensor(rows, dtype=torch.int32)


def plain_move_tokens(k, v, k_dst, v_dst, keep, n, num_kv_heads, mass=None):
    for src, dst in ((k, k_dst), (v, v_dst)):
        was = src.pool.clone()
        for r, ids in enumerate(keep.tolist()):
            for i, j in enumerate(ids):
                dst.pool[int(dst.page_table[r, i // 64]), i % 64] = was[int(src.page_table[r, j // 64]), j % 64]
    return torch.stack([m[ids.long()] for m, ids in zip(mass, keep)])


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(ops.KV, "paged", staticmethod(Plain))
    monkeypatch.setattr(ops, "heavy_tokens", plain_heavy_tokens)
    monkeypatch.setattr(ops, "move_tokens", plain_move_tokens)


def positions(c):
    """The position that every slot of every row holds (each token's key is its position)."""
    return c.k_hf()[:, :, :, 0].float().reshape(c.rows, -1)


def append(c, n):
    at = torch.arange(c.position, c.position + n).to(torch.bfloat16)  # (exact below 256, and in steps of 2 below 512)
    x = at[None, :, None, None].expand(c.batch, n, c.num_kv_heads, 128)
    c.append_tokens(x, x)


def consistent(c):
    mapped = c._pt[c._pt >= 0]
    count = np.bincount(mapped, minlength=c.pool.num_pages)
    assert np.array_equal(count, c.pool.refs) and np.array_equal(c.page_table.numpy(), c._pt)
    assert sorted(c.pool._free) == np.nonzero(count == 0)[0].tolist()


def cache(n, **kw):
    c = PagedKVCache(1, 2, 640, "cpu", with_kmean=False, with_mass=True, **kw)
    append(c, n)
    c.mass[:, :n] = torch.rand((c.rows, n), generator=torch.Generator().manual_seed(n))
    return c


def test_slots_that_an_eviction_picked_stay_picked(plain):
    """A second eviction whose recent tokens reach back into what the first one picked."""
    c = cache(200)
    assert c.evict(128) == 72
    append(c, 10)
    assert c.evict(64, recent=64) == 74  # 54 of the 64 are picked ones, 10 follow the sequence
    assert torch.equal(positions(c)[:, 54:], torch.arange(200.0, 210.0).expand(2, 10))
    with pytest.raises(ValueError, match="before 54 were picked"):
        c.truncate(30)
    with pytest.raises(ValueError, match="before 54 were picked"):
        c.truncate(53)
    c.truncate(55)
    assert c.position == 201 and (positions(c)[:, 54] == 200).all()
    consistent(c)


@pytest.mark.parametrize("first,more,budget,recent", [(0, 10, 60, 8), (30, 5, 90, 35), (30, 5, 90, 36), (64, 1, 100, 100), (100, 60, 64, 64)])
def test_slots_that_follow_the_sequence_after_two_evictions(plain, first, more, budget, recent):
    c = cache(180)
    c.evict(128, recent=first)
    append(c, more)
    c.evict(budget, recent=recent)
    follows = min(recent, first + more)
    assert c._in_order_from == budget - follows
    want = torch.arange(float(c.position - follows), float(c.position))
    assert torch.equal(positions(c)[:, c.length - follows:], want.expand(2, follows))
    consistent(c)
