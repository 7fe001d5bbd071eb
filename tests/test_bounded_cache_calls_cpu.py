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


def models():
    from compactattention_amd.prefill_sparse.llama.modeling_llama_flashprefill_compactattn import LlamaFlashPrefillCompactAttnAttention
    from compactattention_amd.prefill_sparse.llama.modeling_llama_seerattn_chunked_dense import LlamaSeerAttentionChunkedDense

    return {"flash": LlamaFlashPrefillCompactAttnAttention, "seer": LlamaSeerAttentionChunkedDense}


@pytest.mark.parametrize("model,held,tokens,message", [
    ("flash", 100, 200, "at most 64 tokens"), ("seer", 100, 65, "at most 64 tokens"),  # decoded tokens left it inside a block
    ("flash", 192, 128, "multiple of 128 tokens"), ("seer", 128, 64, "gate-K summaries are missing"),
])
@pytest.mark.parametrize("windows", [[0], [0, 2], []])
def test_a_refused_call_leaves_every_layer_as_it_was(model, held, tokens, message, windows):
    """Layer 0 raises before it appends, also where it is under a window itself and another layer refuses."""
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import ChunkedPrefillCache

    kw = dict(sliding_window=40, sliding_window_layers=windows) if windows else {}
    config = SeerAttnLlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=128, num_hidden_layers=3, num_attention_heads=2,
                                 num_key_value_heads=1, **kw)
    config.validate()
    attn = models()[model](config, 0)
    caches = ChunkedPrefillCache(config, 1, 512, "cpu", with_kmean=model == "flash", with_kgate=model == "seer")
    for layer in caches.layers:
        x = torch.zeros((1, held, 1, 128), dtype=torch.bfloat16)
        layer.append_tokens(x, x)
    before = [(c.length, c.position, c._pt.copy(), c.pool.refs.copy()) for c in caches.layers]
    cos = torch.zeros((tokens, 128))
    blocks = torch.zeros((8, 128))
    with pytest.raises(ValueError, match=message):
        attn(torch.zeros((1, tokens, 256), dtype=torch.bfloat16), (cos, cos), past_key_value=caches, block_position_embeddings=(blocks, blocks))
    for c, (length, position, pt, refs) in zip(caches.layers, before):
        assert (c.length, c.position) == (length, position)
        assert np.array_equal(c._pt, pt) and np.array_equal(c.pool.refs, refs)
    assert caches.get_seq_length() == held


def test_calls_that_no_layer_refuses():
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import ChunkedPrefillCache

    kw = dict(vocab_size=64, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1)
    for extra in (dict(), dict(sliding_window=40, sliding_window_layers=[0])):
        caches = ChunkedPrefillCache(SeerAttnLlamaConfig(**kw, **extra), 1, 512, "cpu", with_kmean=True, with_kgate=False)
        for held, calls in ((0, (1, 2, 64, 300)), (100, (1, 64)), (128, (1, 2, 300)), (192, (1,))):
            for layer in caches.layers:
                x = torch.zeros((1, held - layer.length, 1, 128), dtype=torch.bfloat16)
                layer.append_tokens(x, x)
            for tokens in calls:
                caches.check_step(tokens)
    caches = ChunkedPrefillCache(SeerAttnLlamaConfig(**kw, sliding_window=40), 1, 512, "cpu", with_kmean=True, with_kgate=False)
    for layer in caches.layers:
        x = torch.zeros((1, 100, 1, 128), dtype=torch.bfloat16)
        layer.append_tokens(x, x)
    caches.check_step(300)  # windows alone
    caches = ChunkedPrefillCache(SeerAttnLlamaConfig(**kw, seerattn_chunked_prefill_force_dense=True), 1, 512, "cpu", with_kmean=False,
                                 with_kgate=True)
    for layer in caches.layers:
        x = torch.zeros((1, 192, 1, 128), dtype=torch.bfloat16)
        layer.append_tokens(x, x)
    caches.check_step(64)  # chunks that do not select


def test_the_check_of_a_call_counts_the_eviction_before_it(monkeypatch):
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import ChunkedPrefillCache

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    config = SeerAttnLlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2,
                                 num_key_value_heads=1, kv_budget=128)
    caches = ChunkedPrefillCache(config, 1, 512, "cpu", with_kmean=True, with_kgate=False)
    for held, refused in ((150, True), (192, True), (193, False), (300, False)):
        for layer in caches.layers:
            x = torch.zeros((1, held - layer.length, 1, 128), dtype=torch.bfloat16)
            layer.append_tokens(x, x)
        if refused:
            with pytest.raises(ValueError):
                caches.check_step(100)
        else:
            caches.check_step(100)


@pytest.mark.parametrize("settings,recent", [(dict(), 64), (dict(kv_budget_recent=0), 0), (dict(kv_budget_sinks=100), 28),
                                             (dict(kv_budget_sinks=128), 0), (dict(kv_budget=1024, kv_budget_recent=500), 500)])
def test_recent_tokens_that_a_budget_keeps(settings, recent):
    """Tokens just decoded have had few queries: where the setting says nothing, the last ones stay whatever their weights."""
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig

    config = SeerAttnLlamaConfig(**{"kv_budget": 128, **settings})
    config.validate()
    assert config.budget_recent() == recent
    again = SeerAttnLlamaConfig.from_dict(config.to_dict())
    assert again.budget_recent() == recent
    with pytest.raises(ValueError, match="kv_budget"):
        SeerAttnLlamaConfig(kv_budget=128, kv_budget_sinks=129).validate()


def test_a_layer_evicts_with_its_settings(plain, monkeypatch):
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import keep_budget

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = cache(200)
    c.mass[:, 136:] = 0  # decoded tokens without a query yet
    keep_budget(SeerAttnLlamaConfig(kv_budget=128, kv_budget_slack=72), c)
    assert c.length == 200
    keep_budget(SeerAttnLlamaConfig(kv_budget=128, kv_budget_slack=71), c)
    assert c.length == 128 and torch.equal(positions(c)[:, 64:], torch.arange(136.0, 200.0).expand(2, 64))
    assert torch.equal(positions(c)[:, :4], torch.arange(4.0).expand(2, 4))


def budget_caches(max_tokens, **kw):
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import ChunkedPrefillCache

    config = SeerAttnLlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=128, num_hidden_layers=1, num_attention_heads=2,
                                 num_key_value_heads=2, **{"kv_budget": 256, **kw})
    config.validate()
    return config, ChunkedPrefillCache(config, 1, max_tokens, "cpu", with_kmean=False, with_kgate=False)


@pytest.mark.parametrize("budget,slack,max_tokens,slots", [(256, 64, 131072, 256 + 64 + 2048 + 256), (256, 0, 1000, 1024 + 256), (256, 100, 356, 384 + 256),
                                                           (256, 64, 320, 320), (256, 64, 8192, 256 + 64 + 2048 + 256),
                                                           (1024, 8192, 4096, 4096), (4096, 70, 131072, 6272 + 4096)])
def test_a_layer_with_a_budget_holds_pages_for_it(budget, slack, max_tokens, slots):
    """Not for the sequence: budget, slack, a chunk of 2048 and the pages that an eviction moves the budget into."""
    _, caches = budget_caches(max_tokens, kv_budget=budget, kv_budget_slack=slack)
    c = caches.layer(0)
    assert c.cap == slots // 64 and c.pool.num_pages == 2 * (slots // 64) and c.mass.shape == (2, slots)
    assert c.pool.free_pages == 0 and (c._pt >= 0).all()


def test_a_long_run_with_a_budget_takes_no_more_pages(plain, monkeypatch):
    from compactattention_amd.prefill_sparse.llama.modeling_llama_common import keep_budget

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    config, caches = budget_caches(131072)
    c = caches.layer(0)
    pages, cap = c.pool.num_pages, c.cap
    g = torch.Generator().manual_seed(0)
    for n in [2048, 2048, 2048, 700, 1, 64, 2048] + [1] * 70 + [64] * 6 + [2048, 300, 21, 64, 2048]:
        keep_budget(config, c)
        x = torch.randn((1, n, 2, 128), generator=g).to(torch.bfloat16)
        c.append_tokens(x, x)
        c.mass[:, :c.length] += torch.rand((2, c.length), generator=g)
        consistent(c)
    assert (c.pool.num_pages, c.cap) == (pages, cap) and c.position > 5 * 2048
    keep_budget(config, c)
    assert c.length == 256
    c.reset(keep_pages=True)
    consistent(c)
    assert c.pool.num_pages == pages


# reserved: pages behind the tokens (none, some of those that move, all)
@pytest.mark.parametrize("where,reserved", [("alloc", 0), ("alloc", 320), ("pool", 0), ("pool", 320), ("move", 0), ("move", 320), ("move", 640)])
def test_an_eviction_without_memory_leaves_the_cache_as_it_was(plain, monkeypatch, where, reserved):
    c = PagedKVCache(1, 2, 640, "cpu", with_kmean=False, with_mass=True, pool_pages=8)
    append(c, 250)
    c.mass[:, :250] = torch.rand((2, 250), generator=torch.Generator().manual_seed(1))
    if reserved:
        c.reserve(reserved)

    def out_of_memory(*a, **kw):
        raise torch.OutOfMemoryError("none left")

    old = (c.length, c.position, c._pt.copy(), c.pool.refs.copy(), c.mass.clone(), c.k_hf().clone())
    with monkeypatch.context() as m:
        if where == "alloc":
            m.setattr(c.pool, "alloc", out_of_memory)
        elif where == "pool":  # the second of a larger pool's two tensors
            real, calls = c.pool._pages, []
            m.setattr(c.pool, "_pages", lambda n: calls.append(n) or (real(n) if len(calls) == 1 else out_of_memory()))
            c.pool._free, free = [], c.pool._free
        else:
            m.setattr(ops, "move_tokens", out_of_memory)
        with pytest.raises(torch.OutOfMemoryError):
            c.evict(190)
        if where == "pool":
            c.pool._free = free
    assert (c.length, c.position) == old[:2] and np.array_equal(c._pt, old[2]) and torch.equal(c.mass, old[4])
    assert np.array_equal(c.pool.refs[:old[3].size], old[3]) and (c.pool.refs[old[3].size:] == 0).all()
    assert c.pool.k.shape == c.pool.v.shape and torch.equal(c.k_hf(), old[5])
    consistent(c)
    assert c.evict(190) == 60
    consistent(c)


@pytest.mark.parametrize("fails", [1, 2, 3])
def test_tables_and_weights_that_cannot_grow_stay(monkeypatch, fails):
    """The page table on the device, the mean keys and the weights grow together."""
    c = PagedKVCache(1, 2, 64, "cpu", with_mass=True)
    full, zeros, calls = torch.full, torch.zeros, []

    def counted(real):
        def make(*a, **kw):
            calls.append(1)
            if len(calls) == fails:
                raise torch.OutOfMemoryError("none left")
            return real(*a, **kw)
        return make

    with monkeypatch.context() as m:
        m.setattr(torch, "full", counted(full))
        m.setattr(torch, "zeros", counted(zeros))
        with pytest.raises(torch.OutOfMemoryError):
            c.reserve(320)
    assert c.cap == 1 and c._pt.shape == (2, 1) and c.page_table.shape == (2, 1)
    assert c.kmean.shape[2] == 1 and c.mass.shape == (2, 64)
    c.reserve(320)
    assert c.cap == 5 and c.page_table.shape == (2, 5) and c.kmean.shape[2] == 5 and c.mass.shape == (2, 320)


@pytest.mark.parametrize("sinks", [0, 70])
def test_sequences_under_a_window_start_again_in_the_same_pages(sinks):
    """Pages that a window has left behind leave those of its end mapped far from the start, where a new sequence begins."""
    window, chunk = 200, 300
    blocks = -(-sinks // 64) + (window + chunk) // 64 + 3
    c = PagedKVCache(2, 2, 4096, "cpu", with_kmean=False, pool_pages=4 * blocks)
    for _ in range(3):
        for n in [chunk] * 9 + [1] * 5 + [64, 1]:
            x = torch.zeros((2, n, 2, 128), dtype=torch.bfloat16)
            c.append_tokens(x, x)
            c.drop_outside(window, sinks, slack=64)
        assert c.pool.num_pages == 4 * blocks
        used = c.pool.refs.sum()
        c.reset(keep_pages=True)
        consistent(c)
        assert c.pool.refs.sum() == used and (c._pt[:, :used // 4] >= 0).all()
    c.fork(0, 1)
    x = torch.zeros((2, 900, 2, 128), dtype=torch.bfloat16)
    c.append_tokens(x, x)
    c.drop_outside(window, sinks)
    c.fork(0, 1)  # pages that two requests share go back
    c.reset(keep_pages=True)
    consistent(c)
    assert c.pool.refs.max() <= 1
