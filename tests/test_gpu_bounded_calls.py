"""Calls on models and caches of bounded size one after the other: refused calls, rejected drafts, the weights that steer what stays."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd.chunked_prefill import synthetic_prompt
from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM,
                                                       SeerAttnLlamaFlashPrefillCompactAttnForCausalLM)
from tests.test_gpu_bounded_cache import check_pool
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
