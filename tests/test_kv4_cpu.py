"""The 4-bit cache, page copies and the q/k norm without a GPU: the format's oracle against its definition, the
C-ABI's refusals (checked before any launch) and those of the tensor front end."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from compactattention_amd import _hip, ops
from tests import kv4_oracle as ref

FAKE = 1 << 20  # aligned, never dereferenced: validation fails first
INVALID, LIMIT, WORKSPACE = _hip.CA_ERR_INVALID, _hip.CA_ERR_LIMIT, _hip.CA_ERR_WORKSPACE


def _dims(**kw):
    d = dict(batch=1, q_len=4, num_q_heads=8, num_kv_heads=2, kv_cap=10)
    d.update(kw)
    return _hip.Dims(d["batch"], d["q_len"], d["num_q_heads"], d["num_kv_heads"], d["kv_cap"])


def _seq(data=FAKE, sb=0, st=1024, sh=128):
    return _hip.SeqLayout(data, sb, st, sh)


def _kv4(data=FAKE, stride=4352, table=FAKE, pts=16, pages=100):
    return _hip.Kv4Layout(data, stride, table, pts, pages)


def _ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


BAD_KV = [(dict(data=None), INVALID), (dict(data=FAKE + 8), INVALID), (dict(stride=4336), INVALID),
          (dict(stride=4360), INVALID), (dict(table=None), INVALID), (dict(table=FAKE + 2), INVALID),
          (dict(pts=0), INVALID), (dict(pages=0), INVALID), (dict(pages=1 << 31), INVALID)]


def test_format_oracle():
    """Levels, ties, the largest magnitude's bracket and the scale's limits."""
    assert [ref.LEVELS[c] for c in range(8)] == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    x = np.zeros((1, 128))
    x[0, :8] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]  # amax 6: scale 1
    code, byte = ref.quantise(x)
    assert byte[0, 0] == 127 and code[0, :8].tolist() == [7, 0, 2, 2, 4, 4, 6, 6]
    assert byte[0, 1] == 2 and not code[0, 32:].any()
    for top, want in ((7.0, 127), (7.0625, 128), (3.5, 126), (3.53125, 127), (2.0 ** -140, 2), (3.3e38, 252)):
        y = np.zeros((1, 128))
        y[0, 40] = -top
        assert ref.quantise(y)[1][0, 1] == want, top
    rng = np.random.default_rng(0)
    z = ref.bf16(rng.standard_normal((50, 128)) * 10.0 ** rng.integers(-8, 8, (50, 1)))
    code, byte = ref.quantise(z)
    back = ref.values(code, byte)
    top = np.abs(z).reshape(50, 4, 32).max(-1)
    assert ((top / 2.0 ** (byte.astype(float) - 127) <= 7) & (top / 2.0 ** (byte.astype(float) - 127) > 3.5)).all()
    assert (np.abs(back - z) <= 2.0 ** (byte.astype(float) - 127).repeat(32, -1)).all()
    seen = set()
    for of_v in (False, True):
        at = [ref.code_at(t, d, of_v) for t in range(64) for d in range(0, 128, 2)]
        sat = [ref.scale_at(t, g, of_v) for t in range(64) for g in range(4)]
        assert sorted(at) == list(range(4096)) and sorted(sat) == list(range(4096, 4352))
        seen.add(tuple(at))
    assert len(seen) == 2


@pytest.mark.parametrize("kw,code", BAD_KV)
def test_4bit_layouts_are_checked(kw, code):
    lib, d, good, bad = _hip.lib(), _dims(), _kv4(), _kv4(**kw)
    for k, v in ((bad, good), (good, bad)):
        p = [ctypes.byref(x) for x in (d, _seq(), k, v)]
        assert lib.ca_append_q4(p[0], p[1], p[1], p[2], p[3], _ints(0), None) == code
        assert lib.ca_gather_q4(p[0], p[2], p[3], _ints(0), FAKE, FAKE, None) == code
        assert lib.ca_attn_fwd_q4(p[0], p[1], p[2], p[3], FAKE, 16, FAKE, _ints(0), 0.1, p[1], None, 1, None, 0, None) == code
        assert lib.ca_attn_decode_q4(p[0], p[1], p[2], p[3], _ints(64), 0.1, p[1], None, 1, None, 0, None) == code
    assert lib.ca_append_q4(ctypes.byref(d), ctypes.byref(_seq()), ctypes.byref(_seq()), None, ctypes.byref(good), _ints(0), None) == INVALID


@pytest.mark.parametrize("dims,start,code", [
    (dict(batch=0), (0,), INVALID), (dict(batch=65), (0,) * 65, LIMIT), (dict(q_len=0), (0,), INVALID),
    (dict(num_kv_heads=0), (0,), INVALID), (dict(kv_cap=0), (0,), INVALID), (dict(kv_cap=(1 << 24) + 1), (0,), LIMIT),
    (dict(), (-1,), INVALID), (dict(), (637,), INVALID), (dict(batch=2), (0, 640), INVALID),
    (dict(), (2 ** 31 - 1,), INVALID), (dict(q_len=1 << 20, num_kv_heads=1 << 12, kv_cap=1 << 24), (0,), LIMIT),
])
def test_append_and_gather_rows_are_checked(dims, start, code):
    lib, d, kv, s = _hip.lib(), _dims(**dims), _kv4(pts=1 << 25), _seq()
    r = [ctypes.byref(x) for x in (d, s, kv)]
    assert lib.ca_append_q4(r[0], r[1], r[1], r[2], r[2], _ints(*start), None) == code
    assert lib.ca_gather_q4(r[0], r[2], r[2], _ints(*start), FAKE, FAKE, None) == code
    assert lib.ca_append_q4(None, r[1], r[1], r[2], r[2], _ints(*start), None) == INVALID
    assert lib.ca_append_q4(r[0], r[1], r[1], r[2], r[2], None, None) == INVALID


def test_gather_outputs_are_checked():
    lib, d, kv = _hip.lib(), _dims(), _kv4()
    r = [ctypes.byref(x) for x in (d, kv)]
    assert lib.ca_gather_q4(r[0], r[1], r[1], _ints(0), None, FAKE, None) == INVALID
    assert lib.ca_gather_q4(r[0], r[1], r[1], _ints(0), FAKE, None, None) == INVALID
    assert lib.ca_gather_q4(r[0], r[1], None, _ints(0), FAKE, FAKE, None) == INVALID
    assert lib.ca_gather_q4(r[0], r[1], r[1], _ints(0), FAKE + 8, FAKE, None) == INVALID


def test_attention_arguments_are_checked():
    lib = _hip.lib()

    def fwd(dims=None, q=None, table=FAKE, stride=16, counts=FAKE, past=(0,), scale=0.1, splits=1, ws=None, wsb=0):
        r = [ctypes.byref(x) for x in (_dims(**(dims or {})), q or _seq(), _kv4())]
        return lib.ca_attn_fwd_q4(r[0], r[1], r[2], r[2], table, stride, counts, _ints(*past), scale, ctypes.byref(_seq()),
                                  None, splits, ws, wsb, None)

    def decode(dims=None, lens=(64,), scale=0.1, splits=1, ws=None, wsb=0):
        r = [ctypes.byref(x) for x in (_dims(**(dims or {})), _seq(), _kv4())]
        return lib.ca_attn_decode_q4(r[0], r[1], r[2], r[2], _ints(*lens), scale, r[1], None, splits, ws, wsb, None)

    assert fwd(dims=dict(num_q_heads=7)) == INVALID
    assert fwd(dims=dict(num_q_heads=34)) == LIMIT
    assert fwd(dims=dict(kv_cap=0)) == INVALID
    assert fwd(past=(10,)) == INVALID and fwd(past=(-1,)) == INVALID
    assert fwd(q=_seq(data=FAKE + 2)) == INVALID and fwd(q=_seq(st=1023)) == INVALID
    assert fwd(table=None) == INVALID and fwd(counts=None) == INVALID and fwd(stride=9) == INVALID
    assert fwd(table=FAKE + 2) == INVALID and fwd(counts=FAKE + 1) == INVALID
    assert fwd(scale=0.0) == INVALID and fwd(scale=math.nan) == INVALID
    assert fwd(splits=17) == INVALID and fwd(splits=-1) == INVALID and fwd(splits=2) == WORKSPACE
    need = lib.ca_attn_fwd_q4_workspace_size(ctypes.byref(_dims()), _ints(0), 2)
    assert need == 2 * 2 * 4 * 4 * 129 * 4 + 16
    assert lib.ca_attn_fwd_q4_workspace_size(ctypes.byref(_dims()), _ints(0), 17) < 0
    assert lib.ca_attn_decode_q4_workspace_size(ctypes.byref(_dims()), _ints(64), 65) < 0
    assert lib.ca_attn_decode_q4_workspace_size(ctypes.byref(_dims()), _ints(3), 0) < 0
    assert fwd(splits=2, ws=FAKE, wsb=need - 1) == WORKSPACE and fwd(splits=2, ws=FAKE + 4, wsb=need) == WORKSPACE
    assert decode(dims=dict(q_len=65), lens=(65,)) == INVALID
    assert decode(lens=(3,)) == INVALID and decode(lens=(641,)) == INVALID
    assert decode(scale=-1.0) == INVALID and decode(splits=65) == INVALID and decode(splits=2) == WORKSPACE


def test_copy_pages_arguments_are_checked():
    lib = _hip.lib()
    pool = lambda data=FAKE, page=4352, stride=4352, n=10: _hip.PagePool(data, page, stride, n)  # noqa: E731

    def copy(pools, src=(0,), dst=(1,), n=None, ids=None):
        arr = (_hip.PagePool * max(1, len(pools)))(*pools)
        return lib.ca_copy_pages(arr, len(pools), _ints(*src), _ints(*dst), len(src) if n is None else n, ids, None)

    assert copy([]) == INVALID and copy([pool()] * 9) == INVALID
    assert lib.ca_copy_pages(None, 1, _ints(0), _ints(1), 1, None, None) == INVALID
    assert copy([pool(data=None)]) == INVALID and copy([pool(data=FAKE + 8)]) == INVALID
    assert copy([pool(page=0)]) == INVALID and copy([pool(page=4360, stride=4368)]) == INVALID
    assert copy([pool(stride=4336)]) == INVALID and copy([pool(stride=4360)]) == INVALID
    assert copy([pool(page=(1 << 22) + 16, stride=1 << 23)]) == LIMIT
    assert copy([pool(n=0)]) == INVALID
    assert copy([pool()], n=-1) == INVALID
    assert copy([pool(), pool(n=5)], src=(0,), dst=(5,)) == INVALID  # every pool has the page
    assert "outside" in _hip.last_error()
    assert copy([pool()], src=(0, 1), dst=(2, 2)) == INVALID and "written twice" in _hip.last_error()
    assert copy([pool()], src=(0, 1), dst=(2, 0)) == INVALID and "read and written" in _hip.last_error()
    assert copy([pool()], src=(-1,), dst=(2,)) == INVALID and copy([pool()], src=(10,), dst=(2,)) == INVALID
    assert copy([pool()], n=0) == _hip.CA_OK
    assert copy([pool()], ids=FAKE + 2) == INVALID
    assert copy([pool(page=1 << 22, stride=1 << 22, n=1 << 17)], src=[0] * 40000, dst=list(range(1, 40001))) == LIMIT
    assert lib.ca_copy_pages((_hip.PagePool * 1)(pool()), 1, None, _ints(1), 1, None, None) == INVALID


@pytest.mark.parametrize("pages", [5000, 1 << 17, (1 << 17) + 1, 1 << 24])
def test_copies_of_many_pages_are_checked(pages):
    """The page that is named twice is found wherever it stands, with a byte and with a bit a page."""
    lib = _hip.lib()
    pool = (_hip.PagePool * 1)(_hip.PagePool(FAKE, 16, 16, pages))
    ids = np.random.default_rng(pages).permutation(np.arange(pages - 2, pages - 5000, -1))[:4000].astype(np.int32)
    ids[7] = pages - 1  # the last page there is

    def copy(src, dst):
        src, dst = np.ascontiguousarray(src, np.int32), np.ascontiguousarray(dst, np.int32)
        return lib.ca_copy_pages(pool, 1, src.ctypes.data, dst.ctypes.data, len(src), None, None), _hip.last_error()

    src, dst = ids[:2000], ids[2000:]
    for at, other in ((1999, 0), (3, 1234), (1234, 1233)):
        d = dst.copy()
        d[at] = d[other]
        assert copy(src, d) == (INVALID, f"page {d[at]} is written twice")
        d = dst.copy()
        d[at] = src[other]
        assert copy(src, d) == (INVALID, f"page {src[other]} is read and written")
    for bad in (pages, -1):
        s = src.copy()
        s[1500] = bad
        assert copy(s, dst) == (INVALID, f"copy 1500: page {bad} to page {dst[1500]} outside [0, {pages})")


def test_norm_rope_arguments_are_checked():
    lib = _hip.lib()

    def call(q=None, k=None, hq=8, hk=2, w=FAKE, batch=1, length=4, cos=FAKE, csb=0, eps=1e-5):
        s = ctypes.byref(_seq())
        return lib.ca_norm_rope_qk(ctypes.byref(q or _seq()), s, hq, w, ctypes.byref(k or _seq()), s, hk, w, batch, length,
                                   cos, FAKE, csb, eps, None)

    assert call(q=_seq(data=FAKE + 2)) == INVALID and call(k=_seq(st=12)) == INVALID
    assert call(hq=0) == INVALID and call(batch=0) == INVALID and call(length=0) == INVALID
    assert call(hq=70000) == LIMIT and call(batch=1 << 16) == LIMIT and call(length=(1 << 22) + 1) == LIMIT
    assert call(w=None) == INVALID and call(w=FAKE + 2) == INVALID and call(cos=None) == INVALID
    assert call(csb=-4) == INVALID and call(csb=6) == INVALID
    assert call(eps=-1.0) == INVALID and call(eps=math.nan) == INVALID


def test_front_end_refuses_host_tensors():
    pool, table = torch.zeros((4, 4352), dtype=torch.uint8), torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.KV4.paged(pool, table)
    x = torch.zeros((1, 1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="4 bits"):
        ops.append_q4(x, x, None, None, 0, 1)
    with pytest.raises(ValueError, match="shape"):
        ops.append_q4(x, x[:, :, :1], None, None, 0, 1)
    with pytest.raises(ValueError, match="4 bits"):
        ops.gather_q4(None, None, 1, 1, 0, 1)
    with pytest.raises(ValueError, match="GPU"):
        ops.copy_pages([torch.zeros(4, 16)], [0], [1])
    w = torch.zeros(128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.norm_rope_qk(x, x, w, w, 1e-5, torch.zeros(1, 128), torch.zeros(1, 128))


def _cpu_cache(batch=2, heads=2, pages=3):
    from compactattention_amd.kv_cache import PagedKVCache

    return PagedKVCache(batch, heads, 128, "cpu", pool_pages=pages)


def _tokens(n, seed, batch=2, heads=2):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((batch, n, heads, 128), generator=g).to(torch.bfloat16)


def test_cache_truncates_and_compacts():
    """Pages behind a length go back; compaction moves the pages in use to the lowest ids, shared ones with all
    their holders, and gives the rest of the pool back; what is stored stays."""
    c = _cpu_cache()
    k = _tokens(300, 0)
    c.append_tokens(k, -k)
    c.truncate(130)
    assert c.length == 130 and (c.page_table.numpy()[:, 3:] == -1).all()
    assert c.pool.free_pages == c.pool.num_pages - 4 * 3
    assert torch.equal(c.k_hf(), k[:, :130].transpose(1, 2))
    c.fork(0, 1)
    k2 = _tokens(2, 1)
    c.append_tokens(k2, k2)  # the shared last block parts
    want_k, want_v = c.k_hf(), c.v_hf()
    pages = c.pool.num_pages
    used = int((c.pool.refs > 0).sum())
    assert used == 2 * 2 + 4 and pages > used
    table = c.page_table.numpy().copy()
    shared = (table[0, 0], table[2, 0])
    assert shared[0] == shared[1]
    c.compact(shrink=False)
    assert c.pool.num_pages == pages and (c.pool.refs[:used] > 0).all() and (c.pool.refs[used:] == 0).all()
    assert torch.equal(c.k_hf(), want_k) and torch.equal(c.v_hf(), want_v)
    c.compact()
    assert c.pool.num_pages == used and c.pool.free_pages == 0 and c.pool.k.shape[0] == used
    assert torch.equal(c.k_hf(), want_k) and torch.equal(c.v_hf(), want_v)
    table = c.page_table.numpy()
    assert np.array_equal(table, c._pt) and table.max() == used - 1 and table[0, 0] == table[2, 0]
    assert c.compact() == 0
    k3 = _tokens(100, 2)  # the pool grows again
    c.append_tokens(k3, k3)
    assert torch.equal(c.k_hf()[:, :, :132], want_k) and torch.equal(c.k_hf()[:, :, 132:], k3.transpose(1, 2))
    c.truncate(0)
    assert c.pool.free_pages == c.pool.num_pages and c.compact() == 0 and c.pool.num_pages == 1
    c.append_tokens(k3, k3)
    assert torch.equal(c.v_hf(), k3.transpose(1, 2))


def test_cache_truncate_keeps_owned_pages_and_refuses():
    c = _cpu_cache()
    k = _tokens(200, 3)
    c.append_tokens(k, k)
    owned = c.page_table.numpy().copy()
    c.kmean_blocks = c.kgate_blocks = 4
    c.truncate(70, keep_pages=True)
    assert c.length == 70 and np.array_equal(c.page_table.numpy(), owned)
    assert (c.kmean_blocks, c.kgate_blocks) == (1, 1)
    c.append_tokens(k[:, :10], k[:, :10])
    assert torch.equal(c.k_hf(), torch.cat([k[:, :70], k[:, :10]], 1).transpose(1, 2))
    c.fork(0, 1)
    c.truncate(64, keep_pages=True)  # block 1 is shared: both rows of every head give it back
    assert (c.page_table.numpy()[:, 1] == -1).all()
    for bad in (-1, 65):
        with pytest.raises(ValueError, match="truncate"):
            c.truncate(bad)


def test_compact_moves_the_last_pages_into_the_gaps():
    from compactattention_amd.kv_cache import PagePool

    pool = PagePool(8, "cpu")
    ids = pool.alloc(8)
    for p in ids:
        pool.k[p], pool.v[p] = float(p), -float(p)
    pool.release([0, 2, 3, 6])
    pool.retain([7])
    new = pool.compact()
    assert new.tolist() == [-1, 1, -1, -1, 0, 2, -1, 3]
    assert pool.k[:, 0, 0].tolist() == [4, 1, 5, 7] and pool.v[:, 5, 9].tolist() == [-4, -1, -5, -7]
    assert pool.refs.tolist() == [1, 1, 1, 2] and pool.free_pages == 0
    assert sorted(pool.alloc(2)) == [4, 5]


def test_cache_bits_are_checked():
    from compactattention_amd.kv_cache import PagedKVCache
    from compactattention_amd.prefill_sparse.llama import (SeerAttnLlamaChunkedDenseForCausalLM, SeerAttnLlamaConfig)

    with pytest.raises(ValueError, match="bits"):
        PagedKVCache(1, 1, 64, "cpu", bits=8)
    c = PagedKVCache(1, 1, 64, "cpu", bits=4)
    assert c.pool.k.shape == (1, 4352) and c.pool.k.dtype == torch.uint8
    x = torch.zeros((1, 1, 1, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        c.append_tokens(x, x)
    assert c.length == 0
    with pytest.raises(ValueError, match="kv_cache_bits"):
        SeerAttnLlamaConfig(kv_cache_bits=8).validate()
    with pytest.raises(ValueError, match="qk_norm"):
        SeerAttnLlamaChunkedDenseForCausalLM(SeerAttnLlamaConfig(
            vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=1,
            num_key_value_heads=1, max_position_embeddings=128, qk_norm=True))


@pytest.mark.parametrize("heads,q_len,kv,expect", [
    ((32, 8), 1, [64], 1), ((32, 8), 1, [1024], 1),  # up to four fours of blocks: whole
    ((32, 8), 1, [2048], 8), ((32, 8), 1, [8192], 32), ((32, 8), 1, [131072], 32),
    ((32, 8), 1, [4096] * 16, 2),    # 128 rows: two splits fill one round of 256 items
    ((32, 8), 1, [1024] * 32, 1),    # as many rows as places
    ((32, 8), 16, [20011], 16),      # 64 rows: two tiles of 32
    ((64, 64), 1, [131072] * 8, 1),  # more rows than places
])
def test_4bit_decode_split_counts(heads, q_len, kv, expect):
    """Read back from the workspace that the plan asks for."""
    d = _dims(batch=len(kv), q_len=q_len, num_q_heads=heads[0], num_kv_heads=heads[1], kv_cap=-(-max(kv) // 64))
    need = _hip.lib().ca_attn_decode_q4_workspace_size(ctypes.byref(d), _ints(*kv), 0)
    rows = len(kv) * heads[0] * q_len
    assert need == (0 if expect == 1 else expect * rows * 129 * 4 + 16)


@pytest.mark.parametrize("heads,chunk,past,expect", [
    ((32, 8), 1024, [1024], 2), ((32, 8), 2048, [512], 1), ((28, 4), 500, [16, 48, 96, 128], 2),
    ((32, 8), 64, [4], 1), ((32, 8), 256, [24], 1), ((32, 8), 256, [256], 8), ((32, 8), 64, [64], 3), ((8, 8), 64, [0], 1), ((1, 1), 1, [0], 1),
    # one request much longer than the rest: splits of one length, one round more than there are tiles
    ((32, 8), 512, [2000] + [10] * 7, 5), ((32, 8), 1024, [500, 10, 10, 10], 3), ((32, 8), 256, [5, 20, 400], 14),
])
def test_4bit_chunk_split_counts(heads, chunk, past, expect):
    d = _dims(batch=len(past), q_len=chunk, num_q_heads=heads[0], num_kv_heads=heads[1], kv_cap=max(past) + -(-chunk // 64))
    need = _hip.lib().ca_attn_fwd_q4_workspace_size(ctypes.byref(d), _ints(*past), 0)
    rows = len(past) * heads[0] * chunk
    assert need == (0 if expect == 1 else expect * rows * 129 * 4 + 16)
