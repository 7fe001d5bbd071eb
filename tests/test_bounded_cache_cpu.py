"""Pages, positions and refusals of caches of bounded size, on a cache in host memory; the models' settings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaConfig


def cache(n, **kw):
    c = PagedKVCache(2, 2, 640, "cpu", with_kmean=False, **kw)
    x = torch.randn((2, n, 2, 128)).to(torch.bfloat16)
    c.append_tokens(x, x)
    return c


def consistent(c):
    mapped = c._pt[c._pt >= 0]
    count = np.bincount(mapped, minlength=c.pool.num_pages)
    return np.array_equal(count, c.pool.refs) and np.array_equal(c.page_table.numpy(), c._pt)


def test_drop_outside_gives_back_what_no_later_query_sees():
    c = cache(600)
    assert c.drop_outside(700, 3) == 0 and c.drop_outside(537, 3) == 0  # sees token 64 on, block 0 is the sinks'
    assert c.drop_outside(100, 3) == (600 - 99) // 64 - 1
    assert c._pt[0, 0] >= 0 and (c._pt[:, 1:7] == -1).all() and (c._pt[:, 7:10] >= 0).all()
    assert consistent(c)
    assert c.drop_outside(100, 3) == 0
    with pytest.raises(ValueError, match="window of 100"):
        c.drop_outside(50, 3)
    with pytest.raises(ValueError, match="sinks in 1 blocks"):
        c.drop_outside(100, 65)
    with pytest.raises(ValueError, match="were dropped"):
        c.k_hf()
    c.truncate(600 - 53)  # a query at 547 sees 448, the first token that is there
    with pytest.raises(ValueError, match="before 448"):
        c.truncate(546)
    c.fork(0, 1)
    assert consistent(c)
    c.reset()
    assert (c.refs if hasattr(c, "refs") else c.pool.refs).sum() == 0
    x = torch.zeros((2, 5, 2, 128), dtype=torch.bfloat16)
    c.append_tokens(x, x)
    assert c.k_hf().shape == (2, 2, 5, 128) and consistent(c)


def test_dropped_pages_stay_dropped():
    c = cache(600, with_mass=True)
    c.drop_outside(100, 3)
    c.reserve(64 * 12)
    assert (c._pt[:, 1:7] == -1).all() and (c._pt[:, 7:12] >= 0).all() and consistent(c)
    with pytest.raises(ValueError, match="were dropped"):  # the weights of keys that are gone
        c.add_mass(torch.zeros((2, 1, 4, 128), dtype=torch.bfloat16), torch.zeros((2, 4, 1)), 0.1)


def test_slack_keeps_what_a_rejected_draft_brings_back():
    c = cache(600)
    c.drop_outside(100, 0, slack=64)
    c.truncate(536)
    for bad in (dict(window=0), dict(window=5, sinks=-1), dict(window=5, slack=-1)):
        with pytest.raises(ValueError):
            c.drop_outside(**bad)


def test_pages_for_an_eviction_come_from_behind_the_tokens_first():
    c = cache(200, with_mass=True)
    c.reserve(64 * 6)
    tail = c._pt[:, 4:6].copy()
    free = c.pool.free_pages
    pages = c._take_pages(3)
    assert np.array_equal(pages[:, :2], tail) and (c._pt[:, 4:6] == -1).all() and c.pool.free_pages == free - 4
    assert len(set(pages.ravel())) == pages.size and not np.isin(pages, c._pt).any()


def test_what_a_cache_cannot_evict():
    with pytest.raises(ValueError, match="with_mass"):
        cache(200).evict(100)
    with pytest.raises(ValueError, match="with_mass"):
        cache(200).add_mass(torch.zeros((2, 1, 4, 128), dtype=torch.bfloat16), torch.zeros((2, 4, 1)), 0.1)
    with pytest.raises(ValueError, match="gate-K"):
        cache(200, with_mass=True, with_kgate=True).evict(100)
    c = cache(300, with_mass=True)
    for bad in ((0, 0, 0), (10, -1, 0), (10, 0, -1), (10, 6, 5)):
        with pytest.raises(ValueError, match="budget"):
            c.evict(*bad)
    with pytest.raises(ValueError, match="400|queries"):
        c.add_mass(torch.zeros((2, 400, 4, 128), dtype=torch.bfloat16), torch.zeros((2, 4, 400)), 0.1)
    assert c.evict(300) == 0 and c.position == 300
    c.drop_outside(64)
    with pytest.raises(ValueError, match="dropped"):
        c.evict(100)


def test_weights_grow_and_go_with_the_tokens():
    c = cache(100, with_mass=True)
    assert c.mass.shape == (4, 640)
    c.mass[:, :100] = 1.0
    x = torch.zeros((2, 700, 2, 128), dtype=torch.bfloat16)
    c.append_tokens(x, x)
    assert c.mass.shape == (4, c.cap * 64) and (c.mass.sum(1) == 100).all()
    c.truncate(40)
    assert (c.mass.sum(1) == 40).all()
    c.mass[:2] = 0
    c.fork(0, 1)
    assert (c.mass == 0).all()


@pytest.mark.parametrize("bad", [dict(sliding_window=-1), dict(sliding_window=5, sliding_window_sinks=-1), dict(sliding_window_layers=[0]),
                                 dict(sliding_window=5, sliding_window_layers=[32]), dict(kv_budget=100), dict(kv_budget=-128), dict(kv_budget=192),
                                 dict(kv_budget=128, kv_budget_sinks=100, kv_budget_recent=29), dict(kv_budget=128, kv_budget_slack=-1),
                                 dict(kv_budget=128, kv_budget_observe=-1)])
def test_settings_refused(bad):
    with pytest.raises(ValueError):
        SeerAttnLlamaConfig(**bad).validate()


def test_settings():
    c = SeerAttnLlamaConfig(sliding_window=100, sliding_window_layers=[1, 3])
    c.validate()
    assert [c.window_of(i) for i in range(4)] == [0, 100, 0, 100]
    assert SeerAttnLlamaConfig(sliding_window=7).window_of(5) == 7 and SeerAttnLlamaConfig().window_of(0) == 0


def test_the_seer_model_refuses_a_budget():
    from compactattention_amd.prefill_sparse.llama import SeerAttnLlamaChunkedDenseForCausalLM

    with pytest.raises(ValueError, match="kv_budget"):
        SeerAttnLlamaChunkedDenseForCausalLM(SeerAttnLlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=128, num_hidden_layers=1,
                                                                 num_attention_heads=2, num_key_value_heads=1, kv_budget=128))
