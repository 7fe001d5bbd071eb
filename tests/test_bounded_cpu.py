"""Window attention, key weights and eviction on the CPU: what their entry points refuse before any launch, the split plan of
a window, and the oracle against a restatement with masks."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from compactattention_amd import _hip, ops
from tests.bounded_oracle import attention, blocks_seen, kept, random_kv, random_q, visible, weights

FAKE = 1 << 20  # a 16-byte aligned address that is never read: validation fails first


def dims(**kw):
    d = dict(batch=2, q_len=5, num_q_heads=8, num_kv_heads=2, kv_cap=20)
    d.update(kw)
    return _hip.Dims(*(d[n] for n in ("batch", "q_len", "num_q_heads", "num_kv_heads", "kv_cap")))


def seq(data=FAKE, sb=8192, st=1024, sh=128):
    return _hip.SeqLayout(data, sb, st, sh)


def kv(data=FAKE, stok=128, table=FAKE, pts=20, pages=50):
    return _hip.KvLayout(data, 0, 0, 8192, stok, table, pts, pages)


def kv4(data=FAKE, stride=4352, table=FAKE, pts=20, pages=50):
    return _hip.Kv4Layout(data, stride, table, pts, pages)


def ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


def refused(rc, code, text):
    assert rc == code and text in _hip.last_error(), (rc, _hip.last_error())


INVALID, LIMIT, WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("change,code,text", [
    (dict(d=dims(batch=0)), INVALID, "batch"), (dict(d=dims(batch=65)), LIMIT, "batch"), (dict(d=dims(q_len=0)), INVALID, "q_len"),
    (dict(d=dims(num_q_heads=7)), INVALID, "num_q_heads"), (dict(d=dims(num_q_heads=34)), LIMIT, "group"),
    (dict(d=dims(kv_cap=0)), INVALID, "kv_cap"), (dict(d=dims(kv_cap=(1 << 24) + 1)), LIMIT, "kv_cap"),
    (dict(start=ints(0, -1)), INVALID, "request 1"), (dict(start=ints(0, 1276)), INVALID, "request 1"),
    (dict(window=0), INVALID, "window"), (dict(window=-5), INVALID, "window"), (dict(sinks=-1), INVALID, "sinks"),
    (dict(q=seq(data=FAKE + 2)), INVALID, "q data"), (dict(out=seq(st=-1024)), INVALID, "out strides"), (dict(q=seq(data=None)), INVALID, "q is NULL"),
    (dict(scale=0.0), INVALID, "scale"), (dict(scale=math.nan), INVALID, "scale"), (dict(scale=math.inf), INVALID, "scale"),
    (dict(splits=65), INVALID, "num_splits"), (dict(splits=-1), INVALID, "num_splits"), (dict(splits=2), WORKSPACE, "workspace"),
    (dict(lse=FAKE + 1), INVALID, "lse"), (dict(d=dims(q_len=1 << 23, kv_cap=1 << 20)), LIMIT, "group too large"),
])
def test_window_refusals(bits4, change, code, text):
    a = dict(d=dims(), q=seq(), out=seq(), start=ints(3, 700), window=100, sinks=4, scale=0.1, lse=None, splits=1)
    a.update(change)
    cache = kv4() if bits4 else kv()
    entry = getattr(_hip.lib(), "ca_attn_window_q4" if bits4 else "ca_attn_window")
    refused(entry(a["d"], a["q"], cache, cache, a["start"], a["window"], a["sinks"], a["scale"], a["out"], a["lse"], a["splits"], None, 0,
                  None), code, text)


def test_a_window_launch_has_less_than_2_32_threads():
    # 2^20 queries of 64 x 2 rows in tiles of 16, which short windows take: 2^23 workgroups of 512
    d = dims(batch=64, q_len=1 << 20, num_q_heads=2, kv_cap=1 << 14)
    refused(_hip.lib().ca_attn_window(d, seq(), kv(pts=1 << 14), kv(pts=1 << 14), ints(*[0] * 64), 1, 0, 0.1, seq(), None, 1, None, 0, None), LIMIT,
            "too many")


@pytest.mark.parametrize("k,text", [(kv(pts=11), "page_table_stride"), (kv(pages=0), "num_pages"), (kv(stok=4), "strides"),
                                    (kv(data=FAKE + 8), "aligned")])
def test_window_cache_refusals(k, text):
    a = (dims(), seq())
    refused(_hip.lib().ca_attn_window(*a, k, kv(), ints(3, 700), 100, 4, 0.1, seq(), None, 1, None, 0, None), INVALID, text)
    refused(_hip.lib().ca_attn_window(*a, kv(), k, ints(3, 700), 100, 4, 0.1, seq(), None, 1, None, 0, None), INVALID, text)


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("change,code,text", [
    (dict(window=-1), INVALID, "window"), (dict(sinks=-1), INVALID, "sinks"), (dict(start=ints(0, 1276)), INVALID, "request 1"),
    (dict(lse=None), INVALID, "required"), (dict(mass=None), INVALID, "required"), (dict(out=None), INVALID, "required"),
    (dict(mass=FAKE + 2), INVALID, "aligned"), (dict(lse_stride=-1), INVALID, "lse stride"), (dict(counts=None), INVALID, "both"),
    (dict(table=None), INVALID, "both"), (dict(table_stride=19), INVALID, "table_stride"), (dict(mass_stride=704), INVALID, "705"),
    (dict(out_stride=704), INVALID, "705"), (dict(out=FAKE, out_stride=800), INVALID, "one stride"),
    (dict(out=FAKE + 4 * 3000), INVALID, "overlap"), (dict(out=FAKE - 4 * 3000), INVALID, "overlap"), (dict(scale=-1.0), INVALID, "scale"),
    (dict(table=FAKE + 2), INVALID, "aligned"),
])
def test_key_mass_refusals(bits4, change, code, text):
    a = dict(lse=FAKE, lse_stride=100, start=ints(3, 700), window=0, sinks=0, table=FAKE, table_stride=20, counts=FAKE, scale=0.1,
             mass=FAKE, mass_stride=1280, out=1 << 24, out_stride=1280)
    a.update(change)
    entry = getattr(_hip.lib(), "ca_key_mass_q4" if bits4 else "ca_key_mass")
    refused(entry(dims(), seq(), kv4() if bits4 else kv(), a["lse"], a["lse_stride"], 50, a["start"], a["window"], a["sinks"], a["table"],
                  a["table_stride"], a["counts"], a["scale"], a["mass"], a["mass_stride"], a["out"], a["out_stride"], None, 0, None), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=0), INVALID, "batch"), (dict(batch=65), LIMIT, "batch"), (dict(H=0), INVALID, "num_kv_heads"), (dict(budget=0), INVALID, "budget"),
    (dict(lens=ints(-1, 5)), INVALID, "len[0]"), (dict(lens=ints(5, (1 << 30) + 1)), LIMIT, "len[1]"), (dict(sinks=-1), INVALID, "sinks"),
    (dict(recent=-1), INVALID, "recent"), (dict(sinks=30, recent=71), INVALID, "budget"), (dict(mass=None), INVALID, "NULL"),
    (dict(keep=FAKE + 1), INVALID, "misaligned"), (dict(mass_stride=499), INVALID, "500"), (dict(keep_stride=99), INVALID, "100"),
    (dict(sinks=(1 << 31) - 1, recent=(1 << 31) - 1), INVALID, "budget"), (dict(H=1 << 22, lens=ints(500, 500)), LIMIT, "too many"),
])
def test_heavy_tokens_refusals(change, code, text):
    a = dict(mass=FAKE, mass_stride=500, batch=2, H=2, lens=ints(500, 20), budget=100, sinks=3, recent=10, keep=1 << 24, keep_stride=100)
    a.update(change)
    refused(_hip.lib().ca_heavy_tokens(a["mass"], a["mass_stride"], a["batch"], a["H"], a["lens"], a["budget"], a["sinks"], a["recent"],
                                       a["keep"], a["keep_stride"], None, 0, None), code, text)


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("change,code,text", [
    (dict(batch=65), LIMIT, "batch"), (dict(n=0), INVALID, "n=0"), (dict(keep=None), INVALID, "keep"), (dict(keep_stride=99), INVALID, "keep_stride"),
    (dict(mass=None), INVALID, "both"), (dict(mass_stride=499), INVALID, "500"), (dict(out_stride=99), INVALID, "100"),
    (dict(src=7), INVALID, "k page_table_stride"), (dict(dst=1), INVALID, "k_dst page_table_stride"), (dict(mass_out=FAKE + 64), INVALID, "overlap"),
])
def test_move_tokens_refusals(bits4, change, code, text):
    a = dict(src=8, dst=2, keep=FAKE, keep_stride=100, batch=2, lens=ints(500, 20), n=100, mass=FAKE, mass_stride=500, mass_out=1 << 24,
             out_stride=100)
    a.update(change)
    make = kv4 if bits4 else kv
    entry = getattr(_hip.lib(), "ca_move_tokens_q4" if bits4 else "ca_move_tokens")
    refused(entry(make(pts=a["src"]), make(pts=20), make(pts=a["dst"]), make(pts=20), a["keep"], a["keep_stride"], a["batch"], 2, a["lens"],
                  a["n"], a["mass"], a["mass_stride"], a["mass_out"], a["out_stride"], None), code, text)


def test_python_entry_points_refuse_cpu_tensors():
    q = torch.zeros((1, 1, 4, 128), dtype=torch.bfloat16)
    mass = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.KV.heads_first(q)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.attn_window(q, None, None, 0, 1, 0, 0.1, 1, 1)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.key_mass(q, None, None, mass, 0, 0.1, 1, 1)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.heavy_tokens(mass, 10, 2, 5)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.move_tokens(None, None, None, None, torch.zeros((2, 5), dtype=torch.int32), 10, 2)
    with pytest.raises(ValueError, match="KV heads"):
        ops.heavy_tokens(mass, 10, 3, 5)


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("q_len,start,window,sinks", [(1, 131071, 1024, 4), (1, 0, 1, 0), (64, 5000, 1 << 30, 0), (2048, 30720, 4096, 64),
                                                      (300, 100, 1, 1 << 30)])
def test_workspace_of_a_window(bits4, q_len, start, window, sinks):
    """The bytes of the plan's own splits are those of that many splits given."""
    lib = _hip.lib()
    size = lib.ca_attn_window_q4_workspace_size if bits4 else lib.ca_attn_window_workspace_size
    d = dims(batch=1, q_len=q_len, kv_cap=3000)
    auto = size(d, ints(start), window, sinks, 0)
    assert auto in [size(d, ints(start), window, sinks, n) for n in range(1, 65)]
    assert size(d, ints(start), window, sinks, 65) == -1


# ---- the oracle ----
@pytest.mark.parametrize("start,L,W,S", [(0, 70, 5, 2), (100, 40, 33, 3), (64, 1, 64, 0), (90, 50, 1, 200)])
def test_oracle_is_masked_attention(start, L, W, S):
    k, v = random_kv(1, 2, start + L, 1)
    q = random_q(1, L, 4, 1, "cpu")
    cache = type("C", (), dict(k=k.double(), v=v.double(), H=2))()
    out, lse, _, _ = attention(q, cache, [start], W, S)
    p = start + torch.arange(L)[:, None]
    j = torch.arange(start + L)[None, :]
    hidden = (j > p) | ((p - j >= W) & (j >= S))
    total = torch.zeros((2, start + L), dtype=torch.float64)
    for h in range(4):
        s = (q[0, :, h].double() @ k[0, h // 2].double().t()) / math.sqrt(128)
        s = s.masked_fill(hidden, -math.inf)
        w = torch.softmax(s, -1)
        assert torch.allclose(out[0, :, h], w @ v[0, h // 2].double(), rtol=1e-12, atol=1e-12)
        assert torch.allclose(lse[0, h], torch.logsumexp(s, -1), rtol=1e-12, atol=1e-12)
        total[h // 2] += w.sum(0)
    got, _ = weights(q, cache, lse, torch.zeros((2, start + L)), [start], W, S)
    assert torch.allclose(got, total, rtol=1e-12, atol=1e-13)
    seen = sorted(set(int(x) // 64 for x in (~hidden).any(0).nonzero()[:, 0]))
    assert blocks_seen(start, L, W, S) == seen
    assert bool(visible(start, torch.tensor([start]), W, S))


def test_oracle_of_kept_tokens():
    m = np.array([1.0, 5.0, math.nan, 5.0, 0.0, 2.0, 9.0], np.float32)
    assert kept(m, 7, 7, 0, 0) == list(range(7))
    assert kept(m, 7, 3, 0, 0) == [1, 3, 6]
    assert kept(m, 7, 2, 0, 0) == [1, 6]  # of equal weights the first
    assert kept(m, 7, 4, 1, 1) == [0, 1, 3, 6]
    assert kept(m, 7, 6, 0, 0) == [0, 1, 3, 4, 5, 6]  # NaN goes first
