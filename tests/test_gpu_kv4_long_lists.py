"""Long block lists of a 4-bit cache, whole and split, where every page that a border touches is visible by itself.

The queries of a test share a sign pattern.  A marked page holds one token whose key has that pattern, so that it weighs
as much as thousands of others, and whose value is 6 in one head dim, another one for every marked page, and 0 elsewhere.
A marked page that is left out, read twice or read in another's place changes its dim of the output by all of it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from compactattention_amd import ops
from tests import kv4_oracle as ref
from tests.test_gpu_kv4 import SCALE, _check, _tables
from tests.test_gpu_kv4_sizes import _big_cache



def _pattern(seed):
    return np.random.default_rng(seed).choice([-1.0, 1.0], 128)


def _queries(gpu, B, L, Hq, seed):
    """+-1/4 by the pattern, so that a marked key (+-4) scores 128 / sqrt(128) = 11.3."""
    return torch.from_numpy(0.25 * _pattern(seed)).to(torch.bfloat16).expand(B, L, Hq, 128).contiguous().to(gpu)


def _mark(K, V, kt, vt, row, blocks, seed):
    """One token of each of a row's blocks (at most 128 of them, each once)."""
    assert len(blocks) == len(set(blocks)) <= 128
    for i, kb in enumerate(blocks):
        t = (29 * i + 7) % 64
        value = np.zeros(128)
        value[i] = 6.0
        for kv, table, x, of_v in ((K, kt, 4.0 * _pattern(seed), False), (V, vt, value, True)):
            page = int(table[row, kb])
            bytes_ = kv.tensor[page].cpu().numpy()
            ref.write_token(bytes_, t, *ref.quantise(x), of_v)
            kv.tensor[page] = torch.from_numpy(bytes_).to(kv.tensor.device)


def _seen(out, b, heads, blocks):
    """Every marked page carries a share of its own (the tests' own premise)."""
    o = out[b, -1, heads].float()
    assert (o[..., :len(blocks)].abs() > 0.02).all()


def test_a_missing_page_shows():
    """The premise on the CPU: with 60 pages marked of 2048, the output without any one of them is off by more than ten
    tolerances, and so is one that counts it twice."""
    pattern = _pattern(1)
    rng = np.random.default_rng(0)
    n = 2048
    k = torch.from_numpy(rng.choice(ref.LEVELS, (n, 128)) * rng.choice([-1, 1], (n, 128)) * 2.0 ** rng.integers(-8, 1, (n, 1)))
    v = torch.from_numpy(rng.choice(ref.LEVELS, (n, 128)) * rng.choice([-1, 1], (n, 128)) * 2.0 ** rng.integers(-8, 1, (n, 1)))
    marked = torch.arange(0, n, 34)[:60]
    k[marked] = torch.from_numpy(4.0 * pattern)
    v[marked] = 6.0 * torch.eye(128, dtype=torch.float64)[:60]
    q = torch.from_numpy(0.25 * pattern)[None]
    # the unmarked tokens stand for 64 times as many
    w = torch.exp((q @ k.t())[0] * SCALE) * 64.0
    w[marked] /= 64.0
    out = (w @ v) / w.sum()
    A, S = (w @ v.abs()) / w.sum(), (q.abs() @ k.abs().t()).amax() * SCALE
    tol = ref.tolerance(out[None], A[None], S[None])[0]
    for i, at in enumerate(marked.tolist()):
        for factor in (0.0, 2.0):
            x = w.clone()
            x[at] *= factor
            assert abs(float(((x @ v) / x.sum() - out)[i])) > 10 * float(tol[i])


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,L", [(32, 1), (16, 16)])
def test_split_borders_of_131072_tokens(gpu, Hq, L):
    print(f"case: decode4 131072 marked heads={Hq}/4 q_len={L}", flush=True)
    H, n = 4, 131072
    nb = n // 64
    K, V, kt, vt = _big_cache(H, nb, gpu, seed=L)
    q = _queries(gpu, 1, L, Hq, seed=3)
    splits = 32
    edges = [e for s in range(splits) for e in (s * nb // splits, (s + 1) * nb // splits - 1)]  # 64 blocks each
    inner = [640 + i for i in range(1, 24)] + list(range(1089, 1120))
    blocks = edges + [b for b in inner if b not in edges]
    for h in range(H):
        _mark(K, V, kt, vt, h, blocks[h % 2:] + blocks[:h % 2], seed=3)
    for num in (0, splits, 7):
        out, lse = ops.attn_decode(q, K, V, [n], SCALE, nb, H, with_lse=True, num_splits=num)
        _seen(out, 0, slice(None), blocks)
        _check(out, lse, q, K, V, kt, vt, H, [[list(range(nb))] * H], [n - L], [n])


PAGES = (512, 513, 1025)  # of a split: a wave has at most 64, 65 and 129


@pytest.mark.gpu
@pytest.mark.parametrize("nb", PAGES)
@pytest.mark.parametrize("Hq,H,L", [(4, 1, 1), (8, 1, 8)])
def test_many_pages_a_wave(gpu, Hq, H, L, nb):
    """One split, so a wave looks up its pages 64 at a time, more than once."""
    print(f"case: decode4 pages a wave={nb / 8} heads={Hq}/{H} q_len={L}", flush=True)
    n = 64 * nb
    K, V, kt, vt = _big_cache(H, nb, gpu, seed=nb)
    q = _queries(gpu, 1, L, Hq, seed=4)
    blocks = [8 * i + w for i in (0, 1, 62, 63, 64, 65, 127, 128) for w in range(8) if 8 * i + w < nb]
    _mark(K, V, kt, vt, 0, blocks, seed=4)
    out, lse = ops.attn_decode(q, K, V, [n], SCALE, nb, H, with_lse=True, num_splits=1)
    _seen(out, 0, slice(None), blocks)
    _check(out, lse, q, K, V, kt, vt, H, [[list(range(nb))]], [n - L], [n])


@pytest.mark.gpu
@pytest.mark.parametrize("entries", PAGES)
def test_many_pages_a_wave_through_lists(gpu, entries):
    print(f"case: chunk4 list of {entries}", flush=True)
    H, Hq, L, past = 1, 4, 33, 1200
    cap = past + 1
    K, V, kt, vt = _big_cache(H, cap, gpu, seed=entries)
    rng = np.random.default_rng(entries)
    ids = rng.permutation(past)[:entries - 1].tolist()
    ids.insert(entries // 2, past)  # the chunk's own block in the middle
    at = [8 * i + w for i in (0, 1, 62, 63, 64, 65, 127, 128) for w in range(8) if 8 * i + w < entries]
    blocks = [ids[e] for e in at if ids[e] != past]
    _mark(K, V, kt, vt, 0, blocks, seed=6)
    q = _queries(gpu, 1, L, Hq, seed=6)
    table, counts = _tables([[ids]], cap, gpu)
    for splits in (1, 0):
        out, lse = ops.attn_fwd(q, K, V, table, counts, [past], SCALE, cap, H, with_lse=True, num_splits=splits)
        _seen(out, 0, slice(None), blocks)
        _check(out, lse, q, K, V, kt, vt, H, [[ids]], [64 * past], [64 * past + L])


RAGGED = [
    # (Hq, Hkv, q_len, lens): one or two long requests among many short ones, rows and tiles near and past 256 and 512
    (32, 8, 1, [20000] + [640 + 7 * b for b in range(31)]), (32, 8, 1, [900] * 20 + [16383] + [64] * 12),
    (8, 8, 1, [30000] + [70 + b for b in range(63)]), (9, 9, 1, [25000] + [64 + b for b in range(62)] + [10000]),
    # several tiles a row: single splits, whole rows (512, with the splits more than are placed one by one) and 513 rows
    (8, 8, 40, [9000] + [64 + b for b in range(63)]), (9, 9, 40, [9000] + [64 + b for b in range(56)]),
    (32, 8, 40, [20000] + [640] * 4), (28, 4, 16, [300, 12000, 64, 65, 9000, 16, 400, 500, 600, 20]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,H,L,lens", RAGGED)
def test_one_long_request_among_short_ones(gpu, Hq, H, L, lens):
    print(f"case: decode4 ragged heads={Hq}/{H} q_len={L} requests={len(lens)} longest={max(lens)}", flush=True)
    B, nb = len(lens), -(-max(lens) // 64)
    K, V, kt, vt = _big_cache(B * H, nb, gpu, seed=B)
    q = _queries(gpu, B, L, Hq, seed=7)
    b = lens.index(max(lens))
    whole = max(lens) // 64 - 1
    blocks = sorted(set(np.linspace(0, whole, 100).astype(int).tolist()))
    for h in range(H):
        _mark(K, V, kt, vt, b * H + h, blocks, seed=7)
    out, lse = ops.attn_decode(q, K, V, lens, SCALE, nb, H, with_lse=True)
    _seen(out, b, slice(None), blocks)
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens, every=3)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,H,L,past", [(32, 8, 40, [700] + [10] * 5), (16, 2, 20, [5, 900, 0, 60] + [1] * 20)])
def test_one_long_list_among_short_ones(gpu, Hq, H, L, past):
    print(f"case: chunk4 ragged small heads={Hq}/{H} chunk={L} requests={len(past)}", flush=True)
    B = len(past)
    cap = max(past) + 1
    K, V, kt, vt = _big_cache(B * H, cap, gpu, seed=B)
    q = _queries(gpu, B, L, Hq, seed=8)
    b = past.index(max(past))
    blocks = sorted(set(np.linspace(0, max(past) - 1, 100).astype(int).tolist()))
    for h in range(H):
        _mark(K, V, kt, vt, b * H + h, blocks, seed=8)
    lists = [[list(range(p + 1))] * H for p in past]
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True)
    _seen(out, b, slice(None), blocks)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past], every=3)
