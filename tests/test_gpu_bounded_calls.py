"""Calls on models and caches of bounded size one after the other: refused calls, rejected drafts, the weights that steer what stays."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd import ops
from compactattention_amd.chunked_prefill import synthetic_prompt
from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM,
                                                       SeerAttnLlamaFlashPrefillCompactAttnForCausalLM)
from tests.bounded_oracle import SCALE, kept, weights
from tests.test_gpu_bounded_cache import _rand, check_pool, held
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
        table[:, :3] = torch.tensor([[0, 1, past // 64]], dtype=torch.int32)
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


def test_weights_of_a_captured_draft(gpu):
    """A graph adds in place at every replay and holds nothing to take back; a draft before it is forgotten."""
    c, base, q, lse, _, _ = drafted(gpu, 16, 130, 9, False)
    with torch.cuda.device(gpu):
        graph = torch.cuda.CUDAGraph()
        before = c.mass.clone()
        with torch.cuda.graph(graph):
            c.add_mass(q, lse, SCALE, draft=True)
        assert c._draft is None and torch.equal(c.mass, before)
        want = before.clone()
        for _ in range(3):
            graph.replay()
            ops.key_mass(q, c.layouts()[0], lse, want, 130, SCALE, c.cap, c.num_kv_heads)
            torch.cuda.synchronize()
            assert torch.equal(c.mass, want)
        c.truncate(130)
        assert torch.equal(c.mass[:, :130], want[:, :130]) and (c.mass[:, 130:] == 0).all()


@pytest.mark.parametrize("bits", [4, 16])
def test_the_weights_of_attention_under_a_window(gpu, bits):
    """Keys that the window hid get none; eviction by them; a draft's taken back."""
    B, H, Hq, W, S = 2, 2, 8, 70, 5
    g = torch.Generator().manual_seed(bits)
    c = PagedKVCache(B, H, 512, gpu, bits=bits, with_mass=True, with_kmean=False)
    for L in (150, 1, 9, 1):
        start = c.append_tokens(_rand(g, gpu, B, L, H, 128), _rand(g, gpu, B, L, H, 128))
        q = _rand(g, gpu, B, L, Hq, 128)
        _, lse = ops.attn_window(q, *c.layouts(), start, W, S, SCALE, c.cap, H, with_lse=True)
        before, n = c.mass.clone(), c.length
        c.add_mass(q, lse, SCALE, window=W, sinks=S, draft=L == 9)
        want, tol = weights(q, held(c), lse, before[:, :n], [start] * B, W, S)
        assert ((c.mass[:, :n].double().cpu() - want).abs() <= tol).all()
        if start >= S + W:
            assert torch.equal(c.mass[:, S:start - W + 1], before[:, S:start - W + 1])
        if L == 9:
            c.truncate(start + 4)
            want, tol = weights(q[:, :4], held(c), lse[:, :, :4], before[:, :start + 4], [start] * B, W, S)
            assert ((c.mass[:, :start + 4].double().cpu() - want).abs() <= tol).all()
    w, n = c.mass.cpu().numpy().copy(), c.length
    c.evict(100, S, W)
    for r in range(B * H):
        assert torch.equal(c.mass[r, :100].cpu(), torch.from_numpy(w[r])[kept(w[r], n, 100, S, W)])
    with pytest.raises(ops._hip.CaError, match="window"):
        c.add_mass(q[:, :1], lse[:, :, :1], SCALE, window=-1)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dense", [False, True])
def test_the_weights_of_a_model_and_what_it_keeps(gpu, bits, dense, monkeypatch):
    """Every call's weights against 64 bits on the cache's own keys, over the queries, log-sum-exps and lists of the attention itself;
    every eviction against the weights; a rejected draft."""
    m = model_of(FLASH, gpu, kv_budget=256, kv_budget_sinks=4, kv_budget_recent=30, kv_budget_slack=20, kv_budget_observe=50,
                 kv_cache_bits=bits, seerattn_chunked_prefill_force_dense=dense, seerattn_flashprefill_block_size=64,
                 seerattn_flashprefill_alpha=0.9, seerattn_flashprefill_attention_sink=0, seerattn_flashprefill_window_size=1,
                 seerattn_flashprefill_last_n_block=0)
    with torch.no_grad():
        for layer in m.model.layers:  # block scores that differ
            layer.self_attn.q_proj.weight.mul_(8)
            layer.self_attn.k_proj.weight.mul_(8)
    seen = {"attention": None, "votes": 0, "evictions": 0, "listed": 0, "last": {}}
    reals = {n: getattr(ops, n) for n in ("attn_fwd", "attn_decode")}

    def attention(name):
        def call(q, K, V, *a, **kw):
            out, lse = reals[name](q, K, V, *a, **kw)
            seen["attention"] = (q, lse, a[0] if name == "attn_fwd" else None, a[1] if name == "attn_fwd" else None)
            return out, lse
        return call

    add, evict = PagedKVCache.add_mass, PagedKVCache.evict

    def add_mass(self, q, lse, scale, table=None, counts=None, draft=False):
        L, n, before = q.shape[1], self.length, self.mass.clone()
        add(self, q, lse, scale, table, counts, draft)
        aq, alse, atable, acounts = seen["attention"]
        assert L == min(aq.shape[1], 50) and torch.equal(q, aq[:, -L:]) and torch.equal(lse, alse[:, :, -L:])
        lists = None
        if table is not None:
            assert torch.equal(table, atable) and torch.equal(counts, acounts)
            lists = [table[r, :counts[r]].tolist() for r in range(self.rows)]
            seen["listed"] += any(len(x) < -(-n // 64) for x in lists)
        start = [n - L] * self.batch
        want, tol = weights(q, held(self), lse, before[:, :n], start, 0, 0, lists=lists, scale=scale)
        assert ((self.mass[:, :n].double().cpu() - want).abs() <= tol).all() and (self.mass[:, n:] == 0).all()
        # a query's weights over the keys that it saw are a softmax: the sums of a KV head are its group's queries (the
        # log-sum-exp is that of weights rounded to bf16, off by 2^-8 at most)
        votes = L * m.config.num_key_value_groups
        sums = (self.mass - before)[:, :n].double().sum(1).cpu()
        slack = 2.0 ** -24 * self.mass[:, :n].double().sum(1).cpu() + tol.sum(1)
        assert ((sums - votes).abs() <= votes * 2.0 ** -8 + slack).all()
        seen["votes"] += 1
        seen["last"][id(self)] = (before, q, lse, scale, lists, n - L)

    def evicts(self, budget, sinks=0, recent=0, keep_pages=False):
        n, k, v, w = self.length, self.k_hf().clone(), self.v_hf().clone(), self.mass.cpu().numpy().copy()
        assert n > 256 + 20 and (budget, sinks, recent) == (256, 4, 30)
        gone = evict(self, budget, sinks, recent, keep_pages)
        for r in range(self.rows):
            ids = torch.tensor(kept(w[r], n, budget, sinks, recent), device=gpu)
            b, h = divmod(r, self.num_kv_heads)
            assert torch.equal(self.k_hf()[b, h], k[b, h, ids]) and torch.equal(self.v_hf()[b, h], v[b, h, ids])
            assert torch.equal(self.mass[r, :budget].cpu(), torch.from_numpy(w[r])[ids.cpu()])
        seen["evictions"] += 1
        return gone

    for name in reals:
        monkeypatch.setattr(ops, name, attention(name))
    monkeypatch.setattr(PagedKVCache, "add_mass", add_mass)
    monkeypatch.setattr(PagedKVCache, "evict", evicts)
    ids = synthetic_prompt(1, 1280, m.config.vocab_size, 9, gpu)
    cache = m.new_cache(1, 1280)
    m(ids[:, :256], cache)
    for a in range(256, 768, 64):  # (one query block each, so lists leave blocks out)
        m(ids[:, a:a + 64], cache)
    for t in range(768, 794):
        m(ids[:, t:t + 1], cache)
    # drafts, inside a block and past budget and slack: of 7 tokens 2 stay, of 9 none
    for draft, stays in ((7, 2), (9, 0)):
        at = cache.get_seq_length()
        m(ids[:, at:at + draft], cache)
        cache.truncate(at + stays)
        for c in cache.layers:
            before, q, lse, scale, lists, start = seen["last"][id(c)]
            n = start + stays
            want, tol = before[:, :n].double().cpu(), torch.zeros((c.rows, n))
            if stays:
                want, tol = weights(q[:, :stays], held(c), lse[:, :, :stays], before[:, :n], [start], 0, 0, lists=lists, scale=scale)
            assert c.length == n and ((c.mass[:, :n].double().cpu() - want).abs() <= tol).all() and (c.mass[:, n:] == 0).all()
    m(ids[:, 900:901], cache)
    assert seen["votes"] == 2 * (9 + 26 + 2 + 1) and seen["evictions"] >= 2 * 2 and (seen["listed"] > 0) == (not dense)
