"""Caches of bounded size as they are used: weights from chunks and decode steps, eviction, windows whose pages go back, and models
with both."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from compactattention_amd import ops
from compactattention_amd.chunked_prefill import run_chunked_prefill_once, synthetic_prompt
from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM,
                                                       SeerAttnLlamaFlashPrefillCompactAttnForCausalLM)
from tests.bounded_oracle import SCALE, attention, kept, visible, weights
from tests.test_gpu_model import CHUNK, T, tiny_config

pytestmark = pytest.mark.gpu


def _rand(g, gpu, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16).to(gpu)


def held(cache):
    """The cache's own values as the oracle takes them."""
    return type("Held", (), dict(k=cache.k_hf().double().cpu(), v=cache.v_hf().double().cpu(), H=cache.num_kv_heads))()


def check_pool(cache):
    """Every page is mapped as often as it is counted, free pages nowhere; the device's table is the host's."""
    mapped = cache._pt[cache._pt >= 0]
    count = np.bincount(mapped, minlength=cache.pool.num_pages)
    assert np.array_equal(count, cache.pool.refs)
    assert sorted(cache.pool._free) == np.nonzero(count == 0)[0].tolist()
    assert np.array_equal(cache.page_table.cpu().numpy(), cache._pt)


def step(cache, q):
    out, lse = ops.attn_decode(q, *cache.layouts(), [cache.length] * cache.batch, SCALE, cache.cap, cache.num_kv_heads, with_lse=True)
    ref, rlse, tol, ltol = attention(q, held(cache), [cache.length - q.shape[1]] * cache.batch, 1 << 30, 0)
    assert ((out.double().cpu() - ref).abs() <= tol).all() and ((lse.double().cpu() - rlse).abs() <= ltol).all()
    before = cache.mass.clone()
    cache.add_mass(q, lse, SCALE)
    want, mtol = weights(q, held(cache), lse, before, [cache.length - q.shape[1]] * cache.batch, 0, 0)
    n = cache.length
    assert ((cache.mass.cpu().double() - want).abs()[:, :n] <= mtol[:, :n]).all() and (cache.mass[:, n:] == 0).all()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("keep_pages", [False, True])
def test_a_cache_that_evicts(gpu, bits, keep_pages):
    B, H, Hq, budget, sinks, recent = 2, 2, 8, 150, 3, 40
    g = torch.Generator().manual_seed(bits)
    c = PagedKVCache(B, H, 128, gpu, pool_pages=5, bits=bits, with_mass=True)  # the pool, table and weights grow
    # a chunk, whose last queries vote over the blocks of its table
    c.append(_rand(g, gpu, B, 320, H, 128), _rand(g, gpu, B, 320, H, 128))
    q = _rand(g, gpu, B, 320, Hq, 128)
    table, counts = ops.dense_table([0] * B, 320, Hq, H, c.cap, gpu)
    _, lse = ops.attn_fwd(q, *c.layouts(), table, counts, [0] * B, SCALE, c.cap, H, with_lse=True)
    c.add_mass(q[:, -50:], lse[:, :, -50:], SCALE, table, counts)
    want, tol = weights(q[:, -50:], held(c), lse[:, :, -50:], torch.zeros((B * H, 320)), [270] * B, 0, 0)
    assert ((c.mass.cpu().double()[:, :320] - want).abs() <= tol).all()
    c.append_tokens(_rand(g, gpu, B, 3, H, 128), _rand(g, gpu, B, 3, H, 128))
    step(c, _rand(g, gpu, B, 3, Hq, 128))
    c.fork(0, 1)
    assert torch.equal(c.mass[:H], c.mass[H:])
    check_pool(c)
    for n in (323, budget + 70):
        assert c.length == n
        k, v, m = c.k_hf().clone(), c.v_hf().clone(), c.mass.cpu().numpy().copy()
        was = c.position
        assert c.evict(budget, sinks, recent, keep_pages) == n - budget
        assert (c.length, c.position) == (budget, was)
        check_pool(c)
        for r in range(B * H):
            ids = torch.tensor(kept(m[r], n, budget, sinks, recent), device=gpu)
            b, h = divmod(r, H)
            assert torch.equal(c.k_hf()[b, h], k[b, h, ids]) and torch.equal(c.v_hf()[b, h], v[b, h, ids])
            assert np.array_equal(c.mass[r, :budget].cpu().numpy(), m[r, ids.cpu().numpy()])
        assert (c.mass[:, budget:] == 0).all()
        assert c.evict(budget, sinks, recent) == 0
        c.append_tokens(_rand(g, gpu, B, 70, H, 128), _rand(g, gpu, B, 70, H, 128))
        step(c, _rand(g, gpu, B, 9, Hq, 128))
        check_pool(c)
    # a rejected draft into the recent tokens, and no further
    c.truncate(budget - recent)
    assert (c.mass[:, budget - recent:] == 0).all()
    with pytest.raises(ValueError, match="picked by eviction"):
        c.truncate(budget - recent - 1)
    # mean-K of a cache that evicted are those of the keys that it holds
    c.append_tokens(_rand(g, gpu, B, 18, H, 128), _rand(g, gpu, B, 18, H, 128))
    assert c.length == 128
    c.append(_rand(g, gpu, B, 64, H, 128), _rand(g, gpu, B, 64, H, 128))
    mean = c.k_hf().float().view(B, H, 3, 64, 128).mean(3)
    assert ((c.kmean[:, :, :2] - mean[:, :, :2]).abs() <= 64 * 2.0 ** -24 * c.k_hf().float().abs().max()).all()
    c.reset()
    assert (c.length, c.position) == (0, 0) and (c.mass == 0).all()
    check_pool(c)


@pytest.mark.parametrize("bits", [4, 16])
def test_a_cache_under_a_window(gpu, bits):
    B, H, Hq, W, S = 2, 2, 8, 200, 70
    g = torch.Generator().manual_seed(bits + 1)
    c = PagedKVCache(B, H, 1024, gpu, pool_pages=8, bits=bits, with_kmean=False)
    full = PagedKVCache(B, H, 1024, gpu, bits=bits, with_kmean=False)
    most = 0
    for n in (300, 1, 7, 1, 130, 64, 1, 200, 1):
        k, v = _rand(g, gpu, B, n, H, 128), _rand(g, gpu, B, n, H, 128)
        start = c.append_tokens(k, v)
        full.append_tokens(k, v)
        q = _rand(g, gpu, B, n, Hq, 128)
        out = ops.attn_window(q, *c.layouts(), start, W, S, SCALE, c.cap, H)
        assert torch.equal(out, ops.attn_window(q, *full.layouts(), start, W, S, SCALE, full.cap, H))
        ref, _, tol, _ = attention(q, held(full), [start] * B, W, S)
        assert ((out.double().cpu() - ref).abs() <= tol).all()
        c.drop_outside(W, S, slack=64)
        check_pool(c)
        most = max(most, int((c._pt[0] >= 0).sum()))
    assert most <= 2 + (W + 64 + 300) // 64 + 2 and int((c._pt[0] >= 0).sum()) < int((full._pt[0] >= 0).sum())
    c.truncate(c.length - 64)
    with pytest.raises(ValueError, match="were dropped"):
        c.truncate(c.length - 200)
    with pytest.raises(ValueError, match="dropped"):
        c.k_hf()
    with pytest.raises(ValueError, match="window of 200"):
        c.drop_outside(W + 1, S)
    c.fork(0, 1)
    check_pool(c)
    c.compact()
    check_pool(c)


def _run(m, ids, cache, steps):
    logits, _ = run_chunked_prefill_once(m, ids[:, :T], CHUNK, cache)
    out = [logits]
    for i in range(steps):
        out.append(m(ids[:, T + i:T + i + 1], cache))
    return torch.cat(out, 1).float()


@pytest.mark.parametrize("cls", [SeerAttnLlamaChunkedDenseForCausalLM, SeerAttnLlamaFlashPrefillCompactAttnForCausalLM])
@pytest.mark.parametrize("bits", [4, 16])
def test_models_under_a_window(gpu, cls, bits, monkeypatch):
    """Layer 0 under a window: every call of the operator against 64 bits on what was appended to its cache."""
    W, S = 100, 5
    m = cls(tiny_config(kv_cache_bits=bits, sliding_window=W, sliding_window_sinks=S, sliding_window_layers=[0]), device=gpu)
    m.init_weights(seed=11)
    ids = synthetic_prompt(1, T + 40, m.config.vocab_size, 5, gpu)
    cache = m.new_cache(1, T + 64)
    real, calls = ops.attn_window, []

    def window(q, K, V, start, *a, **kw):
        out = real(q, K, V, start, *a, **kw)
        c = cache.layer(0)
        n = c.length
        seen = visible(start, torch.arange(n), W, S)
        seen[max(0, start - W + 1):] = True
        at = seen.nonzero()[:, 0]
        H, held_ = c.num_kv_heads, type("Held", (), dict(H=c.num_kv_heads))()
        for name, pool, of_v in (("k", c.pool.k, False), ("v", c.pool.v, True)):
            full = torch.zeros((1, H, n, 128), dtype=torch.float64)
            for h in range(H):
                pages = torch.from_numpy(c._pt[h][(at // 64).numpy()].astype(np.int64))
                assert (pages >= 0).all()
                if bits == 4:
                    from tests import kv4_oracle
                    full[0, h, at] = kv4_oracle.read_pages(pool.cpu()[pages], of_v)[torch.arange(at.numel()), at % 64]
                else:
                    full[0, h, at] = pool.cpu()[pages, at % 64].double()
            setattr(held_, name, full)
        last = min(q.shape[1], 8)  # the last queries of a chunk
        ref, _, tol, _ = attention(q[:, -last:], held_, [n - last], W, S, scale=a[2])
        assert ((out[:, -last:].double().cpu() - ref).abs() <= tol).all()
        calls.append(q.shape[1])
        return out

    monkeypatch.setattr(ops, "attn_window", window)
    a = _run(m, ids, cache, 3)
    m(torch.flip(ids[:, :17], [1]), cache)  # a draft, rejected
    cache.truncate(T + 3)
    b = m(ids[:, T + 3:T + 4], cache)
    assert calls == [CHUNK] * (T // CHUNK) + [1, 1, 1, 17, 1]
    assert torch.isfinite(a).all() and torch.isfinite(b).all()
    assert cache.layer(0)._dropped[1] > cache.layer(0)._dropped[0] and cache.get_seq_length() == T + 4
    monkeypatch.setattr(ops, "attn_window", real)
    assert torch.equal(_run(m, ids, cache, 3), a)  # a second run in the same cache


def test_a_window_over_everything_is_dense_attention(gpu):
    kw = dict(seerattn_chunked_prefill_force_dense=True)
    out = []
    for extra in ({}, dict(sliding_window=1 << 20, sliding_window_sinks=4)):
        m = SeerAttnLlamaFlashPrefillCompactAttnForCausalLM(tiny_config(**kw, **extra), device=gpu)
        m.init_weights(seed=3)
        ids = synthetic_prompt(1, T + 4, m.config.vocab_size, 6, gpu)
        out.append(_run(m, ids, m.new_cache(1, T + 64), 3))
    assert F.cosine_similarity(out[0].flatten(), out[1].flatten(), dim=0).item() > 0.9999


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dense", [False, True])
def test_models_with_a_budget(gpu, bits, dense):
    cls = SeerAttnLlamaFlashPrefillCompactAttnForCausalLM
    kw = dict(kv_cache_bits=bits, seerattn_chunked_prefill_force_dense=dense)
    plain = cls(tiny_config(**kw), device=gpu)
    plain.init_weights(seed=11)
    ids = synthetic_prompt(2, T + 100, plain.config.vocab_size, 9, gpu)
    want = _run(plain, ids, plain.new_cache(2, T + 128), 4)
    # a budget that nothing reaches changes nothing
    wide = cls(tiny_config(kv_budget=128 * ((T + 300) // 128), **kw), device=gpu)
    wide.init_weights(seed=11)
    assert torch.equal(_run(wide, ids, wide.new_cache(2, T + 128), 4), want)
    m = cls(tiny_config(kv_budget=256, kv_budget_sinks=4, kv_budget_recent=100, kv_budget_slack=20, **kw), device=gpu)
    m.init_weights(seed=11)
    cache = m.new_cache(2, T + 128)
    a = _run(m, ids, cache, 50)
    assert torch.isfinite(a).all()
    for c in cache.layers:
        assert 256 <= c.length <= 256 + 20 and c.position == T + 50
        check_pool(c)
        # each step gives every KV head weights that add up to its query heads (the lse's rounding of 2^-8 aside)
        assert (c.mass[:, :c.length] >= 0).all() and (c.mass[:, c.length:] == 0).all()
    cache.truncate(T + 45)
    assert cache.get_seq_length() == T + 45 and torch.isfinite(m(ids[:, T + 45:T + 46], cache)).all()
    assert torch.equal(_run(m, ids, cache, 50), a)


def test_hf_replacement_with_a_window_and_a_budget(gpu):
    transformers = pytest.importorskip("transformers")
    from compactattention_amd.load_attention_replacement import load_llama_attention_replacement_model, new_compactattn_cache

    cfg = transformers.LlamaConfig(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=128, max_position_embeddings=2048)
    torch.manual_seed(0)
    stock = transformers.LlamaForCausalLM(cfg).to(torch.bfloat16).to(gpu)
    model = load_llama_attention_replacement_model(base_model=stock, variant="flashprefill_compactattn", sliding_window=128,
                                                   sliding_window_sinks=4, sliding_window_layers=[1], kv_budget=128,
                                                   kv_budget_recent=64)
    cache = new_compactattn_cache(model, 1, 640)
    ids = synthetic_prompt(1, 520, 256, 3, gpu)
    with torch.no_grad():
        for a in range(0, 512, 128):
            out = model(input_ids=ids[:, a:a + 128], past_key_values=cache, use_cache=True, logits_to_keep=1).logits
        for a in range(512, 520):
            out = model(input_ids=ids[:, a:a + 1], past_key_values=cache, use_cache=True, logits_to_keep=1).logits
    assert torch.isfinite(out).all() and cache.get_seq_length() == 520
    assert cache.layer(0).length <= 128 + 64 and cache.layer(0).position == 520 and cache.layer(1).length == 520
