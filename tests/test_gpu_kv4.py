"""A KV cache held in 4 bits on the GPU: appends byte for byte and reads value for value against the 64-bit oracle,
attention of single tokens, drafts and chunks within derived tolerances, at the sizes and masks where they can go wrong."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from compactattention_amd import ops
from tests import kv4_oracle as ref

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)


def _table(rows, width, total, seed):
    """Distinct pages in no order."""
    perm = np.random.default_rng(seed).permutation(total)[:rows * width].astype(np.int32)
    return torch.from_numpy(perm.reshape(rows, width))


def _special(L, seed):
    """Tokens [L, 128] whose groups meet every branch of the format."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((L, 4, 32))
    kinds = np.arange(L * 4).reshape(L, 4) % 12
    tops = {1: 7.0, 2: 7.0 * (1 + 2.0 ** -7), 3: 3.5, 4: 2.0 ** -130, 5: 3.3e38, 6: 0.0, 7: 2.0 ** -126}
    for t in range(L):
        for g in range(4):
            k = kinds[t, g]
            if k in tops:
                x[t, g] *= tops[k] / 8
                x[t, g, rng.integers(32)] = tops[k]
            elif k == 8:
                x[t, g] = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -2.5, 6.0], 32)  # ties at scale 1
                x[t, g, 0] = 6.0
            elif k == 9:
                x[t, g, 5] = math.inf
            elif k == 10:
                x[t, g, 31] = math.nan
            elif k == 11:
                x[t, g] *= 1000.0
    return ref.bf16(x.reshape(L, 128))


@pytest.mark.parametrize("B,H,L,starts", [
    (1, 1, 1, [0]), (1, 2, 1, [63]), (2, 2, 1, [64, 5]), (3, 1, 3, [62, 127, 0]), (1, 3, 64, [64]), (1, 2, 65, [1]),
    (2, 4, 130, [37, 300]), (16, 2, 1, [17 * i for i in range(16)]),
])
def test_append_writes_its_bytes_and_no_others(gpu, B, H, L, starts):
    print(f"case: append4 B={B} H={H} L={L} starts={starts}", flush=True)
    width = max(-(-(s + L) // 64) for s in starts)
    total = B * H * width + 5
    rng = np.random.default_rng(B * 1000 + L)
    kt, vt = _table(B * H, width, total, 1), _table(B * H, width, total, 2)
    before = [torch.from_numpy(rng.integers(0, 256, (total, ref.PAGE), dtype=np.uint8)) for _ in range(2)]
    new = [torch.from_numpy(np.stack([_special(L * H, 10 * b + i) for b in range(B)])).view(B, L, H, 128).to(torch.bfloat16)
           for i in range(2)]
    pools = [p.to(gpu) for p in before]
    K, V = ops.KV4.paged(pools[0], kt.to(gpu)), ops.KV4.paged(pools[1], vt.to(gpu))
    # K from a strided view, V contiguous
    wide = torch.zeros((B, L, H + 3, 136), dtype=torch.bfloat16, device=gpu)
    wide[:, :, 1:H + 1, 8:] = new[0].to(gpu)
    ops.append_q4(wide[:, :, 1:H + 1, 8:], new[1].to(gpu), K, V, starts, width)
    back = ops.gather_q4(K, V, B, H, starts, L)
    for i, (pool, table, of_v) in enumerate(((pools[0], kt, False), (pools[1], vt, True))):
        want = before[i].numpy().copy()
        code, byte = ref.quantise(new[i].double().numpy())
        for b in range(B):
            for t in range(L):
                pos = starts[b] + t
                for h in range(H):
                    ref.write_token(want[int(table[b * H + h, pos // 64])], pos % 64, code[b, t, h], byte[b, t, h], of_v)
        assert np.array_equal(pool.cpu().numpy(), want)
        val = torch.from_numpy(ref.values(code, byte)).transpose(1, 2)
        got = back[i].double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(val))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(val))
    only_k, none = ops.gather_q4(K, None, B, H, starts, L)
    assert none is None and torch.equal(torch.nan_to_num(only_k), torch.nan_to_num(back[0]))
    none, only_v = ops.gather_q4(None, V, B, H, starts, L)
    assert none is None and torch.equal(torch.nan_to_num(only_v), torch.nan_to_num(back[1]))


def test_append_skips_pages_outside_the_pool(gpu):
    """A table that names no page (-1, or past the pool): nothing is written for it, and reads are clamped."""
    print("case: append4 bad pages", flush=True)
    pool = torch.full((3, ref.PAGE), 7, dtype=torch.uint8, device=gpu)
    table = torch.tensor([[-1, 1], [2, 3]], dtype=torch.int32, device=gpu)  # row 1's second page does not exist
    K = ops.KV4.paged(pool, table)
    V = ops.KV4.paged(pool.clone(), table)
    x = torch.randn((1, 100, 2, 128), device=gpu).to(torch.bfloat16)
    ops.append_q4(x, x, K, V, 0, 2)
    for kv in (K, V):
        got = kv.tensor.cpu()
        assert (got[0] == 7).all()  # page 0 is where a clamp of -1 would have written
        assert (got[1] != 7).any() and (got[2] != 7).any()
    ops.gather_q4(K, V, 1, 2, 0, 100)
    torch.cuda.synchronize()


def _cache(B, H, blocks, gpu, seed, dtype_scale=1.0):
    """A cache of `blocks` pages a row with tokens quantised in it: (K, V, table on the host)."""
    rng = np.random.default_rng(seed)
    total = B * H * blocks + 3
    pools = []
    for of_v in (False, True):
        x = rng.standard_normal((total, 64, 128)) * dtype_scale
        if not of_v:
            x[..., rng.integers(0, 128, 4)] *= 4
        pools.append(ref.make_pages(torch.from_numpy(ref.bf16(x)), of_v))
    kt, vt = _table(B * H, blocks, total, seed + 1), _table(B * H, blocks, total, seed + 2)
    K = ops.KV4.paged(pools[0].to(gpu), kt.to(gpu))
    V = ops.KV4.paged(pools[1].to(gpu), vt.to(gpu))
    return K, V, kt, vt


def _row(pool, table_row, ids, of_v):
    """fp64 tokens of a row's blocks `ids` (a list)."""
    pages = pool[table_row[torch.as_tensor(ids, dtype=torch.long)].long().to(pool.device)]
    return ref.read_pages(pages, of_v).reshape(-1, 128)


def _check(out, lse, q, K, V, kt, vt, H, lists, qpos0, kv_len, every=1):
    """Every KV row (or every so many) against the oracle.  lists[b][h]: block ids; keys at or past kv_len[b] do not exist."""
    B, L, Hq, _ = q.shape
    G = Hq // H
    for b in range(B):
        for h in range(H):
            r = b * H + h
            if r % every:
                continue
            ids = lists[b][h]
            rows = q[b, :, h * G:(h + 1) * G].reshape(L * G, 128).double()
            qp = (qpos0[b] + torch.arange(L)).repeat_interleave(G).to(q.device)
            if len(ids) == 0:
                k = v = torch.zeros((0, 128), dtype=torch.float64, device=q.device)
                kpos = torch.zeros(0, dtype=torch.long, device=q.device)
            else:
                k, v = _row(K.tensor, kt[r], ids, False), _row(V.tensor, vt[r], ids, True)
                kpos = (64 * torch.as_tensor(ids)[:, None] + torch.arange(64)).reshape(-1).to(q.device)
                there = kpos < kv_len[b]
                k, v, kpos = k[there], v[there], kpos[there]
            want, wlse, A, S = ref.attention(rows, k, v, kpos, qp, SCALE)
            got = out[b, :, h * G:(h + 1) * G].reshape(L * G, 128).double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, h)
            ok = ~torch.isnan(want)
            tol = ref.tolerance(torch.nan_to_num(want), torch.nan_to_num(A), torch.nan_to_num(S))
            err = (got - want).abs()
            assert (err[ok] <= tol[ok]).all(), (b, h, float((err / tol)[ok].max()))
            if lse is not None:
                gl = lse[b, h * G:(h + 1) * G].t().reshape(-1).double()
                assert torch.equal(torch.isnan(gl), torch.isnan(wlse)), (b, h)
                fin = torch.isfinite(wlse)
                assert torch.equal(gl[~fin & ~torch.isnan(wlse)], wlse[~fin & ~torch.isnan(wlse)])
                assert ((gl - wlse).abs()[fin] <= ref.lse_tolerance(S)[fin]).all()


DECODE = [
    # (Hq, Hkv, q_len, lens, splits)
    (1, 1, 1, [1], 0), (8, 2, 1, [63], 0), (8, 2, 1, [64], 0), (8, 2, 1, [65], 0), (32, 8, 1, [1000], 0),
    (28, 4, 1, [129, 1, 64, 777], 0), (16, 1, 1, [300, 4000], 0), (8, 8, 1, [2000], 3), (8, 2, 4, [4, 260, 67], 0),
    (32, 8, 1, [5000], 7), (4, 1, 3, [3], 2), (8, 2, 4, [577], 9),
    # more than 16 packed rows
    (28, 4, 3, [900, 64], 0), (32, 8, 16, [1000], 0), (16, 2, 64, [64, 100, 1337], 0), (8, 8, 40, [40], 0),
    (16, 1, 64, [3000], 5), (24, 6, 9, [72, 9, 513], 3),
]


@pytest.mark.parametrize("Hq,H,L,lens,splits", DECODE)
def test_decode(gpu, Hq, H, L, lens, splits):
    print(f"case: decode4 heads={Hq}/{H} q_len={L} lens={lens} splits={splits}", flush=True)
    B, blocks = len(lens), -(-max(lens) // 64)
    K, V, kt, vt = _cache(B, H, blocks, gpu, seed=L * 7 + max(lens))
    g = torch.Generator().manual_seed(5)
    q = torch.randn((B, L, Hq + 2, 128), generator=g).to(torch.bfloat16).to(gpu)[:, :, 1:Hq + 1]  # strided
    out, lse = ops.attn_decode(q, K, V, lens, SCALE, blocks, H, out=torch.empty((B, L, Hq, 128), dtype=torch.bfloat16, device=gpu),
                               with_lse=True, num_splits=splits)
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)


CHUNK = [
    # (Hq, Hkv, chunk, past blocks, kept share, splits)
    (1, 1, 1, [0], 1.0, 0), (8, 2, 64, [0], 1.0, 0), (8, 2, 100, [3], 0.5, 0), (4, 4, 65, [1, 7], 0.5, 0),
    (28, 4, 130, [5, 0, 20], 0.3, 0), (16, 1, 200, [70], 0.4, 4), (8, 8, 257, [9], 1.0, 2), (32, 8, 64, [140], 0.9, 0),
    (2, 1, 1024, [0], 1.0, 0), (6, 2, 33, [33, 66, 2], 0.7, 3), (16, 2, 31, [300], 0.25, 16),
]


def _lists(B, H, past, qb, keep, seed):
    rng = np.random.default_rng(seed)
    out = []
    for b in range(B):
        rows = []
        for h in range(H):
            kept = np.nonzero(rng.random(past[b]) < keep)[0].tolist()
            rows.append(kept + list(range(past[b], past[b] + qb)))
        out.append(rows)
    return out


def _tables(lists, cap, gpu, pad=3):
    rows = [r for b in lists for r in b]
    table = torch.full((len(rows), cap + pad), 1 << 20, dtype=torch.int32)  # behind the lists: anything
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    return table.to(gpu), torch.tensor([len(r) for r in rows], dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("Hq,H,L,past,keep,splits", CHUNK)
def test_chunk(gpu, Hq, H, L, past, keep, splits):
    print(f"case: chunk4 heads={Hq}/{H} chunk={L} past={past} keep={keep} splits={splits}", flush=True)
    B, qb = len(past), -(-L // 64)
    cap = max(past) + qb
    K, V, kt, vt = _cache(B, H, cap, gpu, seed=L + max(past))
    q = torch.randn((B, L, Hq, 128), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(gpu)
    lists = _lists(B, H, past, qb, keep, seed=L)
    table, counts = _tables(lists, cap, gpu)
    out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [64 * p for p in past], [64 * p + L for p in past])


def test_chunk_rows_without_blocks(gpu):
    """Lists that are empty, or that hold only blocks some queries do not see: zeros and -inf for the rest."""
    print("case: chunk4 empty lists", flush=True)
    B, H, Hq, L, past = 1, 4, 8, 150, [2]
    cap = 5
    K, V, kt, vt = _cache(B, H, cap, gpu, seed=3)
    q = torch.randn((B, L, Hq, 128), generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(gpu)
    lists = [[[], [4], [3, 4], [0]]]
    table, counts = _tables(lists, cap, gpu)
    for splits in (1, 2):
        out, lse = ops.attn_fwd(q, K, V, table, counts, past, SCALE, cap, H, with_lse=True, num_splits=splits)
        _check(out, lse, q, K, V, kt, vt, H, lists, [128], [128 + L])
        assert (out[0, :, 0:2] == 0).all() and torch.isneginf(lse[0, 0:2]).all()
        assert (out[0, :128, 2:4] == 0).all()


def _poison(K, V, table_k, table_v, row, pos, what):
    """NaN groups in the page that holds position pos of a row."""
    for kv, table, of_v, name in ((K, table_k, False, "k"), (V, table_v, True, "v")):
        if name in what:
            page = int(table[row, pos // 64])
            for g in what[name]:
                kv.tensor[page, ref.scale_at(pos % 64, g, of_v)] = 255


@pytest.mark.parametrize("rows16", [True, False])
@pytest.mark.parametrize("splits", [1, 3])
def test_nan_in_hidden_places_of_a_draft(gpu, rows16, splits):
    """Positions at and past kv_len hold NaN: no effect.  A NaN value in the draft reaches the tokens that see it,
    in its dims, and no others; a NaN key all dims."""
    Hq, H, L = (8, 2, 4) if rows16 else (8, 2, 20)
    lens = [64 * 9 + 30, 64 * 3 + 64]
    print(f"case: decode4 nan heads={Hq}/{H} q_len={L} splits={splits}", flush=True)
    B, blocks = 2, 11
    K, V, kt, vt = _cache(B, H, blocks, gpu, seed=40)
    for b in range(B):
        for h in range(H):
            for pos in range(lens[b], min(-(-lens[b] // 64) * 64, lens[b] + 40)):
                _poison(K, V, kt, vt, b * H + h, pos, {"k": range(4), "v": range(4)})
    q = torch.randn((B, L, Hq, 128), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(gpu)
    lists = [[list(range(-(-n // 64)))] * H for n in lens]
    args = (q, K, V, lens, SCALE, blocks, H)
    out, lse = ops.attn_decode(*args, with_lse=True, num_splits=splits)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)
    _poison(K, V, kt, vt, 0, lens[0] - 2, {"v": [1, 3]})  # seen by the last two tokens of row 0
    _poison(K, V, kt, vt, 3, lens[1] - 1, {"k": [2]})     # seen by the last token of row 3
    _poison(K, V, kt, vt, 1, 70, {"v": [0]})              # seen by all, in a block that is not masked
    out, lse = ops.attn_decode(*args, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [n - L for n in lens], lens)
    assert torch.isnan(out[0, L - 1, 0, 32:64]).all() and torch.isfinite(out[0, L - 3, 0]).all()
    assert torch.isnan(out[1, L - 1, 4:]).all() and torch.isfinite(out[1, L - 2, 4:]).all()
    assert torch.isnan(out[0, :, 4:, :32]).all() and torch.isfinite(out[0, :, 4:, 32:]).all()


@pytest.mark.parametrize("splits", [1, 2])
def test_nan_in_hidden_places_of_a_chunk(gpu, splits):
    Hq, H, L, past = 8, 2, 300, [4]
    print(f"case: chunk4 nan splits={splits}", flush=True)
    cap = 4 + 5
    K, V, kt, vt = _cache(1, H, cap, gpu, seed=41)
    for h in range(H):
        for pos in range(256 + L, 64 * cap):
            _poison(K, V, kt, vt, h, pos, {"k": range(4), "v": range(4)})
    lists = [[[0, 2, 4, 5, 6, 7, 8], [1, 4, 5, 6, 7, 8]]]
    for pos in (3 * 64, 3 * 64 + 5):  # in a block that no list names
        _poison(K, V, kt, vt, 0, pos, {"k": range(4), "v": range(4)})
    table, counts = _tables(lists, cap, gpu)
    q = torch.randn((1, L, Hq, 128), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(gpu)
    args = (q, K, V, table, counts, past, SCALE, cap, H)
    out, lse = ops.attn_fwd(*args, with_lse=True, num_splits=splits)
    assert torch.isfinite(out).all()
    _check(out, lse, q, K, V, kt, vt, H, lists, [256], [256 + L])
    _poison(K, V, kt, vt, 0, 256 + 130, {"v": [2]})
    _poison(K, V, kt, vt, 1, 256 + 77, {"k": [0], "v": [0, 1, 2, 3]})
    out, lse = ops.attn_fwd(*args, with_lse=True, num_splits=splits)
    _check(out, lse, q, K, V, kt, vt, H, lists, [256], [256 + L])
    assert torch.isfinite(out[0, :130, :4]).all() and torch.isnan(out[0, 130:, :4, 64:96]).all()
    assert torch.isfinite(out[0, :77, 4:]).all() and torch.isnan(out[0, 77:, 4:]).all()


@pytest.mark.parametrize("spread", [30.0, 0.0])
def test_scores_far_apart(gpu, spread):
    """Scores of hundreds and of nothing at all in one row: one key carries the softmax, or all weigh alike."""
    print(f"case: decode4 extreme scores {spread}", flush=True)
    K, V, kt, vt = _cache(1, 2, 9, gpu, seed=50, dtype_scale=spread)
    q = (torch.randn((1, 1, 8, 128), generator=torch.Generator().manual_seed(3)) * 20).to(torch.bfloat16).to(gpu)
    lists = [[list(range(9))] * 2]
    out, lse = ops.attn_decode(q, K, V, [64 * 9], SCALE, 9, 2, with_lse=True)
    # the scores' error is relative to sums of |q k|, thousands here: the tolerance says so
    _check(out, lse, q, K, V, kt, vt, 2, lists, [64 * 9 - 1], [64 * 9])
    table, counts = _tables([[list(range(9))] * 2], 9, gpu)
    qc = q.expand(1, 64, 8, 128).contiguous()
    out, lse = ops.attn_fwd(qc, K, V, table, counts, [8], SCALE, 9, 2, with_lse=True)
    _check(out, lse, qc, K, V, kt, vt, 2, lists, [512], [576])


def test_pages_past_32_bits(gpu):
    """Pools of more than 4 GiB: pages at their far end are read and written."""
    print("case: 4-bit pools of 4.5 GB", flush=True)
    total = (1 << 32) // ref.PAGE + 200_000
    kt = torch.tensor([[total - 1, 0, total // 2], [total - 3, total - 2, 5]], dtype=torch.int32)
    pools = [torch.zeros((total, ref.PAGE), dtype=torch.uint8, device=gpu) for _ in range(2)]
    K, V = (ops.KV4.paged(p, kt.to(gpu)) for p in pools)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((1, 190, 2, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    ops.append_q4(k.to(gpu), v.to(gpu), K, V, 0, 3)
    for x, back in zip((k, v), ops.gather_q4(K, V, 1, 2, 0, 190)):
        assert torch.equal(back.double().cpu().transpose(1, 2), torch.from_numpy(ref.values(*ref.quantise(x.double().numpy()))))
    q = torch.randn((1, 1, 8, 128), generator=g).to(torch.bfloat16).to(gpu)
    out, lse = ops.attn_decode(q, K, V, [190], SCALE, 3, 2, with_lse=True)
    lists = [[[0, 1, 2]] * 2]
    _check(out, lse, q, K, V, kt, kt, 2, lists, [189], [190])
    table, counts = _tables(lists, 3, gpu)
    qc = torch.randn((1, 62, 8, 128), generator=g).to(torch.bfloat16).to(gpu)
    out, lse = ops.attn_fwd(qc, K, V, table, counts, [2], SCALE, 3, 2, with_lse=True)
    _check(out, lse, qc, K, V, kt, kt, 2, lists, [128], [190])


def test_requests_that_share_pages_read_the_same(gpu):
    """Decode of forked requests (the same pages at the same places, then pages of their own, of different lengths)
    gives bit for bit what the same values on separate pages give: where an item's pages are shared, another copy of
    its code runs."""
    print("case: forks", flush=True)
    B, H, G, blocks = 5, 2, 4, 40
    lens = [64 * 40, 64 * 40 - 13, 64 * 17 + 1, 5, 64 * 33]
    first_own = [0, 30, 12, 0, 20]  # request 0's pages up to here (request 3 shares nothing)
    K, V, kt, vt = _cache(B, H, blocks, gpu, 77)
    shared = []
    for kv, own in ((K, kt), (V, vt)):
        forked = own.clone()
        for b in range(B):
            forked[b * H:(b + 1) * H, :first_own[b]] = own[:H, :first_own[b]]
        shared.append(ops.KV4.paged(kv.tensor, forked.to(gpu)))
        moved = forked != own
        ops.copy_pages(kv.tensor, forked[moved], own[moved])
    torch.manual_seed(5)
    q = torch.randn((B, 1, H * G, 128), device=gpu, dtype=torch.bfloat16)
    for splits in (0, 1, 3):
        a = ops.attn_decode(q, *shared, lens, SCALE, blocks, H, with_lse=True, num_splits=splits)
        b = ops.attn_decode(q, K, V, lens, SCALE, blocks, H, with_lse=True, num_splits=splits)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_pools_with_a_page_stride(gpu):
    """Pages that are a part of larger records, one pool for K and V."""
    print("case: decode4 strided pages", flush=True)
    K, V, kt, vt = _cache(1, 2, 5, gpu, seed=60)
    n = K.tensor.shape[0]
    both = torch.zeros((n, 2 * ref.PAGE + 16), dtype=torch.uint8, device=gpu)
    both[:, :ref.PAGE], both[:, ref.PAGE + 16:] = K.tensor, V.tensor
    K2 = ops.KV4.paged(both[:, :ref.PAGE], K.page_table)
    V2 = ops.KV4.paged(both[:, ref.PAGE + 16:], V.page_table)
    q = torch.randn((1, 2, 4, 128), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(gpu)
    assert torch.equal(ops.attn_decode(q, K, V, [300], SCALE, 5, 2), ops.attn_decode(q, K2, V2, [300], SCALE, 5, 2))
    a, b = ops.gather_q4(K, V, 1, 2, 7, 200), ops.gather_q4(K2, V2, 1, 2, 7, 200)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_results_repeat_and_ride_streams_and_graphs(gpu):
    """The same bits on a second call, on another stream, and from a graph that holds append, decode and chunk."""
    print("case: kv4 graph", flush=True)
    H, Hq, blocks = 2, 8, 12
    K, V, kt, vt = _cache(1, H, blocks, gpu, seed=70)
    g = torch.Generator().manual_seed(4)
    q = torch.randn((1, 1, Hq, 128), generator=g).to(torch.bfloat16).to(gpu)
    qc = torch.randn((1, 128, Hq, 128), generator=g).to(torch.bfloat16).to(gpu)
    kn, vn = (torch.randn((1, 1, H, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    table, counts = _tables([[[0, 3, 5, 10, 11], [2, 10, 11]]], blocks, gpu)

    def step():
        ops.append_q4(kn, vn, K, V, 64 * 12 - 1, blocks)
        a = ops.attn_decode(q, K, V, [64 * 12], SCALE, blocks, H)
        b = ops.attn_fwd(qc, K, V, table, counts, [10], SCALE, blocks, H, num_splits=2)
        return a, b, *ops.gather_q4(K, V, 1, H, 64 * 12 - 1, 1)

    want = [t.clone() for t in step()]
    again = step()
    assert all(torch.equal(x, y) for x, y in zip(want, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for r in range(3):
        q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16))
        kn.copy_(torch.randn(kn.shape, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, got)), r
