"""The operators together, as they are used: a paged cache in 4 bits (and in 16) through chunks, decode steps, a fork, a
rejected draft and compaction, and models on such a cache and with normed queries and keys."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from compactattention_amd import ops
from compactattention_amd.chunked_prefill import run_chunked_prefill_once, synthetic_prompt
from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM,
                                                       SeerAttnLlamaFlashPrefillCompactAttnForCausalLM)
from tests import kv4_oracle as ref
from tests.test_gpu_model import CHUNK, T, tiny_config
from tests.test_gpu_pages_norm import _norm_rope64

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)


def _rand(g, gpu, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16).to(gpu)


def _stored(x, bits):
    """What a cache of these bits stands for: [B, H, n, 128] fp64 on the CPU."""
    x = x.double().cpu().transpose(1, 2)
    return x if bits == 16 else torch.from_numpy(ref.values(*ref.quantise(x.numpy())))


def _attend(cache, q, length, lists=None):
    """The oracle over the cache's own values: (want, tolerance) [L, Hq, 128] of request b."""
    k, v = cache.k_hf().double(), cache.v_hf().double()
    B, L, Hq, _ = q.shape
    H = cache.num_kv_heads
    G = Hq // H
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    for b in range(B):
        for h in range(H):
            kpos = torch.arange(length, device=q.device)
            if lists is not None:
                kpos = (64 * torch.tensor(lists[b][h], device=q.device)[:, None] + torch.arange(64, device=q.device)).reshape(-1)
                kpos = kpos[kpos < length]
            qp = torch.arange(length - L, length, device=q.device).repeat_interleave(G)
            rows = q[b, :, h * G:(h + 1) * G].reshape(L * G, 128).double()
            o, _, A, S = ref.attention(rows, k[b, h, kpos], v[b, h, kpos], kpos, qp, SCALE)
            want[b, :, h * G:(h + 1) * G] = o.view(L, G, 128)
            tol[b, :, h * G:(h + 1) * G] = ref.tolerance(o, A, S).view(L, G, 128)
    return want, tol


@pytest.mark.parametrize("bits", [4, 16])
def test_a_cache_through_its_life(gpu, bits):
    print(f"case: cache life bits={bits}", flush=True)
    B, H, Hq = 2, 2, 8
    g = torch.Generator().manual_seed(bits)
    c = PagedKVCache(B, H, 128, gpu, pool_pages=5, bits=bits)  # the pool, the table and the summaries grow
    ref16 = PagedKVCache(B, H, 128, gpu, pool_pages=5)
    toks = []

    def both(n, op):
        k, v = _rand(g, gpu, B, n, H, 128), _rand(g, gpu, B, n, H, 128)
        toks.append((k, v))
        for x in (c, ref16):
            getattr(x, op)(k, v)

    def check_values():
        for got, i in ((c.k_hf(), 0), (c.v_hf(), 1)):
            want = _stored(torch.cat([t[i] for t in toks], 1), bits)
            assert torch.equal(got.double().cpu(), want)

    for n in (192, 128):
        both(n, "append")
    check_values()
    assert torch.equal(c.kmean[:, :, :5], ref16.kmean[:, :, :5])  # the summaries are of the bf16 keys
    # a selecting chunk, with its query means
    q = _rand(g, gpu, B, 100, Hq, 128)
    k, v = _rand(g, gpu, B, 100, H, 128), _rand(g, gpu, B, 100, H, 128)
    toks.append((k, v))
    past, qhat = c.append_with_query_means(k, v, q)
    past16, qhat16 = ref16.append_with_query_means(k, v, q)
    assert past == past16 == 5 and torch.equal(qhat, qhat16)
    rowmask, _ = ops.score_select(qhat, c.kmean, SCALE, ops.Rule(topk=0, sink_blocks=1, local_blocks=1), [5] * B, H, c.cap)
    table, counts, _, _ = ops.union_compact(rowmask, [5] * B, H, c.cap)
    K, V = c.layouts()
    out = ops.attn_fwd(q, K, V, table, counts, [5] * B, SCALE, c.cap, H)
    lists = [[table[b * H + h, :int(counts[b * H + h])].tolist() for h in range(H)] for b in range(B)]
    assert all(r == [0, 4, 5, 6] for b in lists for r in b)
    want, tol = _attend(c, q, 420, lists)
    assert ((out.double() - want).abs() <= tol).all()
    # decode steps into the partial block, a draft, most of it rejected
    for n in (1, 5, 20):
        both(n, "append_tokens")
    check_values()
    qd = _rand(g, gpu, B, 20, Hq, 128)
    K, V = c.layouts()
    out = ops.attn_decode(qd, K, V, [c.length] * B, SCALE, c.cap, H)
    want, tol = _attend(c, qd, c.length)
    assert ((out.double() - want).abs() <= tol).all()
    for x in (c, ref16):
        x.truncate(428)
    toks[-1] = tuple(t[:, :2] for t in toks[-1])
    check_values()
    # request 1 goes on from request 0's tokens
    for x in (c, ref16):
        x.fork(0, 1)
    for i, t in enumerate(toks):
        toks[i] = tuple(y[:1].expand(B, *y.shape[1:]) for y in t)
    check_values()
    both(3, "append_tokens")
    check_values()
    # compaction: the same bits before and after
    qd = _rand(g, gpu, B, 1, Hq, 128)
    K, V = c.layouts()
    before = ops.attn_decode(qd, K, V, [c.length] * B, SCALE, c.cap, H)
    pages = c.pool.num_pages
    for x in (c, ref16):
        assert x.compact() >= 0
    assert c.pool.num_pages == int((c.pool.refs > 0).sum()) < pages
    check_values()
    K, V = c.layouts()
    assert torch.equal(ops.attn_decode(qd, K, V, [c.length] * B, SCALE, c.cap, H), before)
    # tokens that fill the block: its mean-K is that of the stored keys, and chunks go on
    both(64 * 7 - c.length, "append_tokens")
    c.refresh_kmean(7)
    keys = c.k_hf()[:, :, 384:448].double().mean(2)
    # 64 sums in fp32 and a division: 65 roundings of at most 2^-24 of the sum of magnitudes
    bound = 65 * 2.0 ** -24 * c.k_hf()[:, :, 384:448].double().abs().mean(2) * 1.01
    assert ((c.kmean[:, :, 6].double() - keys).abs() <= bound).all()
    both(64, "append")
    check_values()
    c.reset()
    assert c.length == 0 and c.pool.free_pages == c.pool.num_pages


def test_compaction_moves_many_pages(gpu):
    """Pages scattered over a pool by two interleaved caches' worth of growth; every other one freed."""
    print("case: compact many", flush=True)
    for bits in (4, 16):
        c = PagedKVCache(4, 8, 64, gpu, pool_pages=1, bits=bits)
        g = torch.Generator().manual_seed(1)
        for _ in range(5):
            x = _rand(g, gpu, 4, 64 * 8, 8, 128)
            c.append(x, x)
        c.truncate(64 * 21 + 5)
        k, v = c.k_hf().clone(), c.v_hf().clone()
        used = 32 * 22
        assert c.pool.num_pages > used
        c.compact()
        assert c.pool.num_pages == used
        assert torch.equal(c.k_hf(), k) and torch.equal(c.v_hf(), v)
        # a hole in every row: forks release pages at the front
        c.fork(3, 0)
        k, v = c.k_hf().clone(), c.v_hf().clone()
        moved = c.compact()
        assert moved > 0 and c.pool.num_pages == used - 8 * 22
        assert torch.equal(c.k_hf(), k) and torch.equal(c.v_hf(), v)


@pytest.mark.parametrize("L,past", [(200, 40), (64, 0), (1, 33)])
def test_four_bits_agree_with_bf16_on_the_same_values(gpu, L, past):
    """Attention over the 4-bit pages against the bf16 kernels over the values they stand for."""
    print(f"case: kv4 against bf16 L={L} past={past}", flush=True)
    H, Hq, B = 2, 8, 2
    g = torch.Generator().manual_seed(L)
    n = 64 * past + L
    c = PagedKVCache(B, H, n, gpu, bits=4)
    k, v = _rand(g, gpu, B, n, H, 128), _rand(g, gpu, B, n, H, 128)
    c.append(k, v)
    q = _rand(g, gpu, B, L, Hq, 128)
    K, V = c.layouts()
    K16, V16 = ops.KV.heads_first(c.k_hf()), ops.KV.heads_first(c.v_hf())
    if L == 1:
        a = ops.attn_decode(q, K, V, [n] * B, SCALE, c.cap, H)
        b = ops.attn_decode(q, K16, V16, [n] * B, SCALE, c.cap, H)
    else:
        table, counts = ops.dense_table([past] * B, L, Hq, H, c.cap, gpu)
        a = ops.attn_fwd(q, K, V, table, counts, [past] * B, SCALE, c.cap, H)
        b = ops.attn_fwd(q, K16, V16, table, counts, [past] * B, SCALE, c.cap, H)
    want, tol = _attend(c, q, n)
    assert ((a.double() - want).abs() <= tol).all() and ((b.double() - want).abs() <= tol).all()


def _logits64(model, ids):
    """The model's last logits in 64 bits over the whole prompt, dense, with the q/k norms where it has them."""
    c = model.config
    sd = {k: v.detach().double().cpu() for k, v in model.state_dict().items()}
    L = ids.shape[1]
    cos, sin = (getattr(model.model.rotary_emb, n)[:L].double().cpu() for n in ("cos", "sin"))
    h = sd["model.embed_tokens.weight"][ids.cpu()]
    rms = lambda x, w: w * x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + c.rms_norm_eps)  # noqa: E731
    for i in range(c.num_hidden_layers):
        p = f"model.layers.{i}."
        x = rms(h, sd[p + "input_layernorm.weight"])
        q, k, v = ((x @ sd[p + f"self_attn.{n}_proj.weight"].T).view(1, L, -1, 128) for n in "qkv")
        if c.qk_norm:
            q, k = rms(q, sd[p + "self_attn.q_norm.weight"]), rms(k, sd[p + "self_attn.k_norm.weight"])
        rot = lambda y: y * cos[None, :, None] + torch.cat([-y[..., 64:], y[..., :64]], -1) * sin[None, :, None]  # noqa: E731
        q, k = rot(q), rot(k)
        G = c.num_key_value_groups
        k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) * SCALE
        s = s.masked_fill(torch.ones(L, L, dtype=torch.bool).triu(1), -math.inf)
        o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v).reshape(1, L, -1)
        h = h + o @ sd[p + "self_attn.o_proj.weight"].T
        x = rms(h, sd[p + "post_attention_layernorm.weight"])
        h = h + (F.silu(x @ sd[p + "mlp.gate_proj.weight"].T) * (x @ sd[p + "mlp.up_proj.weight"].T)) @ sd[p + "mlp.down_proj.weight"].T
    return rms(h, sd["model.norm.weight"])[:, -1:] @ sd["lm_head.weight"].T


def _build(cls, gpu, **kw):
    m = cls(tiny_config(**kw), device=gpu)
    m.init_weights(seed=11)
    if kw.get("qk_norm"):
        g = torch.Generator(device=gpu).manual_seed(3)
        with torch.no_grad():
            for layer in m.model.layers:
                for n in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                    assert (n.weight == 1).all()
                    n.weight.uniform_(0.5, 1.5, generator=g)
    return m


def test_model_with_qk_norms(gpu):
    """Dense chunks, a decode step, a draft that is rejected, another step, on a bf16 cache: each step's logits against
    64 bits, as near as the models without norms are held to."""
    print("case: model qk_norm", flush=True)
    m = _build(SeerAttnLlamaFlashPrefillCompactAttnForCausalLM, gpu, seerattn_chunked_prefill_force_dense=True, qk_norm=True)
    ids = synthetic_prompt(1, T + 2, m.config.vocab_size, 4321, gpu)
    cache = m.new_cache(1, T + 64)

    def near(got, n):
        want = _logits64(m, ids[:, :n]).float()
        got = got.float().cpu()
        assert F.cosine_similarity(got.flatten(), want.flatten(), dim=0).item() > 0.999
        assert (got - want).abs().max().item() <= 0.05 * want.abs().max().item()

    near(run_chunked_prefill_once(m, ids[:, :T], CHUNK, cache)[0], T)
    near(m(ids[:, T:T + 1], cache), T + 1)
    m(torch.flip(ids[:, :17], [1]), cache)
    cache.truncate(T + 1)
    cache.compact()
    near(m(ids[:, T + 1:], cache), T + 2)


@pytest.mark.parametrize("cls,qk_norm", [(SeerAttnLlamaChunkedDenseForCausalLM, False),
                                         (SeerAttnLlamaFlashPrefillCompactAttnForCausalLM, True)])
def test_models_on_a_4_bit_cache(gpu, cls, qk_norm, monkeypatch):
    """Every call that a model makes of the operators, against 64 bits on the call's own inputs: what is appended is what
    the format says, and every layer's attention is that of the values in its cache.  (Logits of the two caches are not
    compared: a key next to a rounding border falls on either side of it.)"""
    print(f"case: model kv4 {cls.__name__} qk_norm={qk_norm}", flush=True)
    m = _build(cls, gpu, seerattn_chunked_prefill_force_dense=True, kv_cache_bits=4, qk_norm=qk_norm)
    ids = synthetic_prompt(1, T + 2, m.config.vocab_size, 4321, gpu)
    cache = m.new_cache(1, T + 64)
    assert cache.layer(0).bits == 4
    seen = {"append": 0, "chunk": 0, "decode": 0, "norm": 0}
    real = {n: getattr(ops, n) for n in ("append_q4", "attn_fwd", "attn_decode", "norm_rope_qk")}

    def append(k, v, K, V, start, cap):
        real["append_q4"](k, v, K, V, start, cap)
        back = ops.gather_q4(K, V, k.shape[0], k.shape[2], start, k.shape[1])
        for new, got in zip((k, v), back):
            assert torch.equal(got.double().cpu(), _stored(new, 4))
        seen["append"] += 1

    def holder(K):
        return next(c for c in cache.layers if c.pool.k.data_ptr() == K.tensor.data_ptr())

    def check(out, q, K, length):
        c = holder(K)
        c_len, c.length = c.length, length
        want, tol = _attend(c, q, length)
        c.length = c_len
        assert ((out.double() - want).abs() <= tol).all()

    def chunk(q, K, V, table, counts, past, *a, **kw):
        out = real["attn_fwd"](q, K, V, table, counts, past, *a, **kw)
        check(out, q, K, 64 * past[0] + q.shape[1])
        seen["chunk"] += 1
        return out

    def decode(q, K, V, kv_len, *a, **kw):
        out = real["attn_decode"](q, K, V, kv_len, *a, **kw)
        check(out, q, K, kv_len[0])
        seen["decode"] += 1
        return out

    def norm(q, k, qw, kw, eps, cos, sin):
        got = real["norm_rope_qk"](q, k, qw, kw, eps, cos, sin)
        for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
            want, terms = _norm_rope64(x, w, eps, cos, sin)
            assert ((y.double() - want).abs() <= 1.01 * (75 * 2.0 ** -24 * terms + 2.0 ** -8 * want.abs()) + 2.0 ** -126).all()
        seen["norm"] += 1
        return got

    for n, f in (("append_q4", append), ("attn_fwd", chunk), ("attn_decode", decode), ("norm_rope_qk", norm)):
        monkeypatch.setattr(ops, n, f)
    logits, _ = run_chunked_prefill_once(m, ids[:, :T], CHUNK, cache)
    first = m(ids[:, T:T + 1], cache)
    m(torch.flip(ids[:, :17], [1]), cache)
    cache.truncate(T + 1)
    cache.compact()
    last = m(ids[:, T + 1:], cache)
    for x in (logits, first, last):
        assert torch.isfinite(x).all()
    layers = m.config.num_hidden_layers
    assert seen == {"append": layers * (T // CHUNK + 3), "chunk": layers * (T // CHUNK), "decode": layers * 3,
                    "norm": layers * (T // CHUNK + 3) if qk_norm else 0}


@pytest.mark.parametrize("cls", [SeerAttnLlamaChunkedDenseForCausalLM, SeerAttnLlamaFlashPrefillCompactAttnForCausalLM])
def test_selecting_models_on_a_4_bit_cache(gpu, cls):
    """A selecting prefill and a step; a second run in the same pages gives the same bits."""
    print(f"case: model kv4 selecting {cls.__name__}", flush=True)
    m = cls(tiny_config(kv_cache_bits=4), device=gpu)
    m.init_weights(seed=11)
    ids = synthetic_prompt(2, T + 37, m.config.vocab_size, 77, gpu)
    cache = m.new_cache(2, T)
    a, _ = run_chunked_prefill_once(m, ids, CHUNK, cache)
    step = m(ids[:, :1], cache)
    b, _ = run_chunked_prefill_once(m, ids, CHUNK, cache)
    assert torch.isfinite(a).all() and torch.isfinite(step).all() and torch.equal(a, b)
