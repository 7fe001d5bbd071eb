"""Truncation of a cache whose last chunk ended inside a block: gate-K summaries stay valid while every token that they
pooled stays, and a sequence with rejected drafts goes on as one without."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd.kv_cache import PagedKVCache
from compactattention_amd.synthetic import rope_tables


def _tokens(n, g):
    return torch.randn((1, n, 2, 128), generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("draft,to,blocks", [(5, 100, 2), (5, 104, 2), (0, 100, 2), (60, 101, 2), (5, 99, 1), (5, 64, 1), (5, 63, 0), (5, 0, 0)])
def test_gate_summaries_of_a_truncated_cache(draft, to, blocks):
    g = torch.Generator().manual_seed(draft)
    c = PagedKVCache(1, 2, 256, "cpu", with_kgate=True)
    x = _tokens(100 + draft, g)
    c.append_tokens(x[:, :100], x[:, :100])
    c.kgate_blocks, c.kgate_tokens = 2, 100  # as after a chunk of 100 tokens with its gate
    c.append_tokens(x[:, 100:], x[:, 100:])
    c.truncate(to)
    assert c.kgate_blocks == blocks
    c.truncate(to)
    assert c.kgate_blocks == blocks
    # what is appended behind a cut block does not bring its summary back
    c.append_tokens(x[:, :40], x[:, :40])
    c.truncate(to + 20)
    assert c.kgate_blocks == blocks
    c.reset()
    assert (c.kgate_blocks, c.kgate_tokens) == (0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_a_rejected_draft_does_not_stop_the_next_chunk(gpu, bits):
    print(f"case: rejected draft, bits={bits}", flush=True)
    g = torch.Generator().manual_seed(3)
    wk = (torch.randn((2, 128, 128), generator=g) * 0.02).float().to(gpu)
    cos, sin = (t.to(gpu) for t in rope_tables(8))
    kw = dict(gate_wk=wk, rope_cos=cos, rope_sin=sin)
    first, rest, chunk, draft = (_tokens(n, g).to(gpu) for n in (100, 28, 128, 9))
    plain = PagedKVCache(1, 2, 512, gpu, with_kgate=True, bits=bits)
    drafted = PagedKVCache(1, 2, 512, gpu, with_kgate=True, bits=bits)
    for c in (plain, drafted):
        c.append(first, first, **kw)
        if c is drafted:
            for n in (100, 103, 100):
                c.append_tokens(draft, draft)
                c.truncate(n)
        c.append_tokens(rest, rest)
        assert c.append(chunk, chunk, **kw) == 2
        assert (c.length, c.kmean_blocks, c.kgate_blocks) == (256, 4, 4)
    assert torch.equal(plain.k_hf(), drafted.k_hf()) and torch.equal(plain.v_hf(), drafted.v_hf())
    assert torch.equal(plain.kgate[:, :, :4], drafted.kgate[:, :, :4]) and torch.equal(plain.kmean[:, :, :4], drafted.kmean[:, :, :4])
    drafted.truncate(192)  # the second chunk's last block goes
    assert drafted.kgate_blocks == 3
    assert drafted.append(chunk[:, :64], chunk[:, :64], **kw) == 3
