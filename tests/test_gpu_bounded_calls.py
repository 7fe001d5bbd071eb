"""Calls on models and caches of bounded size one after the other: refused calls, rejected drafts, the weights that steer what stays."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd import ops
from compactattention_amd.chunked_prefill import synthetic_prompt
from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM,
                                                       SeerAttnLlamaFlashPrefillCompactAttnForCausalLM)
from tests.bounded_oracle import SCALE
from tests.test_gpu_bounded_cache import _rand, check_pool
from tests.test_gpu_model import tiny_config

pytestmark = pytest.mark.gpu

FLASH, SEER = SeerAttnLlamaFlashPrefillCompactAttnForCausalLM, SeerAttnLlamaChunkedDenseForCausalLM


def model_of(cls, gpu, seed=11, **kw):
    m = cls(tiny_config(**kw), device=gpu)
    m.init_weights(seed=seed)
    return m


@pytest.mark.parametrize("cls", [FLASH, SEER])
def test_a_refused_turn_can_be_sent_again_in_pieces(gpu, cls):
    """Windows on layer 0 take any number of tokens, layer 1 refuses more than 64 past a prompt of 100."""
    m = model_of(cls, gpu, sliding_window=60, sliding_window_layers=[0])
    ids = synthetic_prompt(1, 300, m.config.vocab_size, 5, gpu)
    out = []
    for refused in (False, True):
        cache = m.new_cache(1, 512)
        m(ids[:, :100], cache)
        if refused:
            before = [(c.length, c._pt.copy()) for c in cache.layers]
            with pytest.raises(ValueError, match="at most 64"):
                m(ids[:, 100:300], cache)
            assert all(c.length == n and (c._pt == pt).all() for c, (n, pt) in zip(cache.layers, before))
            assert cache.get_seq_length() == 100
        for a in range(100, 300, 50):
            logits = m(ids[:, a:a + 50], cache)
        out.append(logits)
        assert [c.length for c in cache.layers] == [300, 300]
        for c in cache.layers:
            check_pool(c)
    assert torch.equal(*out)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("draft", [2, 17, 64])
def test_a_draft_past_the_budget_can_be_rejected(gpu, bits, draft):
    """With the settings' defaults: a draft that takes the cache past budget and slack leaves all its tokens to be rejected, and the
    next call evicts."""
    m = model_of(FLASH, gpu, kv_budget=256, kv_cache_bits=bits)
    ids = synthetic_prompt(2, 512, m.config.vocab_size, 5, gpu)
    cache = m.new_cache(2, 512)
    m(ids[:, :256], cache)
    for t in range(256, 319):
        m(ids[:, t:t + 1], cache)
    m(ids[:, 319:319 + draft], cache)  # (319: inside a block, where more than one token is a draft)
    assert all(c.length == 319 + draft and c.evicted == 0 for c in cache.layers)
    for kept in (draft - 1, 1, 0):
        cache.truncate(319 + kept)
        assert cache.get_seq_length() == 319 + kept
    m(ids[:, 319:319 + draft], cache)
    cache.truncate(321)
    logits = m(ids[:, 321:321 + draft], cache)  # the first call past the budget: it evicts before it appends
    assert torch.isfinite(logits).all() and all(c.length == 256 + draft and c.evicted == 65 for c in cache.layers)
    cache.truncate(321)
    assert all(c.length == 256 for c in cache.layers) and cache.get_seq_length() == 321
    for t in range(321, 500):
        logits = m(ids[:, t:t + 1], cache)
        assert all(256 < c.length <= 256 + 64 + 1 for c in cache.layers)
    assert torch.isfinite(logits).all()
    for c in cache.layers:
        check_pool(c)


def test_a_long_turn_after_an_eviction(gpu):
    """A chunk that starts past the budget starts at it, so also where decoded tokens left the cache inside a block."""
    m = model_of(FLASH, gpu, kv_budget=256)
    ids = synthetic_prompt(1, 1024, m.config.vocab_size, 6, gpu)
    cache = m.new_cache(1, 1024)
    m(ids[:, :300], cache)
    with pytest.raises(ValueError, match="at most 64"):
        m(ids[:, 300:400], cache)  # 300 is within the slack
    m(ids[:, 300:350], cache)
    assert all(c.length == c.position == 350 for c in cache.layers)
    logits = m(ids[:, 350:550], cache)  # evicted to 256, a whole block
    assert torch.isfinite(logits).all() and all(c.length == 256 + 200 and c.position == 550 for c in cache.layers)
    for c in cache.layers:
        check_pool(c)


def drafted(gpu, bits, past, L, lists, draft=True, seed=0):
    """A cache of past tokens with weights, and a draft of L tokens whose queries voted."""
    B, H, Hq = 2, 2, 8
    g = torch.Generator().manual_seed(seed)
    c = PagedKVCache(B, H, 512, gpu, bits=bits, with_mass=True, with_kmean=False)
    c.append_tokens(_rand(g, gpu, B, past, H, 128), _rand(g, gpu, B, past, H, 128))
    c.mass[:, :past] = torch.rand((B * H, past), generator=g).to(gpu)
    base = c.mass.clone()
    c.append_tokens(_rand(g, gpu, B, L, H, 128), _rand(g, gpu, B, L, H, 128))
    q = _rand(g, gpu, B, L, Hq, 128)
    _, lse = ops.attn_decode(q, *c.layouts(), [c.length] * B, SCALE, c.cap, H, with_lse=True)
    table = counts = None
    if lists:
        table = torch.zeros((B * H, c.cap), dtype=torch.int32, device=gpu)
        table[:, :3] = torch.tensor([[0, 2, past // 64]], dtype=torch.int32)
        counts = torch.full((B * H,), 3, dtype=torch.int32, device=gpu)
        counts[1] = 2
    c.add_mass(q, lse, SCALE, table, counts, draft=draft)
    return c, base, q, lse, table, counts


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("past,L,lists", [(200, 20, False), (192, 20, True), (0, 7, False), (250, 64, False)])
def test_the_weights_of_a_rejected_draft_go(gpu, bits, past, L, lists):
    c, base, q, lse, table, counts = drafted(gpu, bits, past, L, lists)
    for stays in (L - 1, 5, 5, 1, 0):
        want = base.clone()
        if stays:
            ops.key_mass(q[:, :stays].clone(), c.layouts()[0], lse[:, :, :stays].clone(), want, past, SCALE, c.cap, c.num_kv_heads,
                         table=table, counts=counts)
        assert (want != base).any() == (stays > 0)
        c.truncate(past + stays)
        assert torch.equal(c.mass, want), stays
    if past:
        c.truncate(past - 5)
        base[:, past - 5:] = 0
        assert torch.equal(c.mass, base)


def test_weights_of_drafts_between_other_calls(gpu):
    L, past = 9, 130
    # several calls back at once; and what is not called a draft stays
    c, base, *_ = drafted(gpu, 16, past, L, False)
    c.truncate(past - 1)
    base[:, past - 1:] = 0
    assert torch.equal(c.mass, base)
    c, base, *_ = drafted(gpu, 16, past, L, False, draft=False)
    after = c.mass.clone()
    c.truncate(past)
    assert torch.equal(c.mass[:, :past], after[:, :past]) and (c.mass[:, past:] == 0).all()
    # tokens appended behind a draft that stays, and rejected
    c, base, q, lse, _, _ = drafted(gpu, 16, past, L, False)
    after = c.mass.clone()
    x = torch.zeros((2, 3, 2, 128), dtype=torch.bfloat16, device=gpu)
    c.append_tokens(x, x)
    c.truncate(past + L)
    assert torch.equal(c.mass, after)
    # a later call's weights are added to those of the draft, which then stay
    c.append_tokens(x, x)
    c.add_mass(q[:, :3], lse[:, :, :3], SCALE)
    after = c.mass.clone()
    c.truncate(past + 2)
    assert torch.equal(c.mass[:, :past + 2], after[:, :past + 2])
    # a fork's weights go with those of the request that it shares
    c, base, *_ = drafted(gpu, 16, past, L, True)
    c.fork(1, 0)
    c.truncate(past + 4)
    one, base, *_ = drafted(gpu, 16, past, L, True)
    one.truncate(past + 4)
    assert torch.equal(c.mass[:2], c.mass[2:]) and torch.equal(c.mass[2:], one.mass[2:])
    # an eviction or a new sequence forgets the draft
    c, base, *_ = drafted(gpu, 16, past, L, False)
    c.evict(100, recent=30)
    mass = c.mass.clone()
    c.truncate(80)
    assert torch.equal(c.mass[:, :80], mass[:, :80])
    c, base, *_ = drafted(gpu, 16, past, L, False)
    c.reset(keep_pages=True)
    c.append_tokens(x, x)
    c.truncate(1)
    assert (c.mass == 0).all()
