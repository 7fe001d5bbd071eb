"""Page copies and the norm of queries and keys with their rotation, on the GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from compactattention_amd import _hip, ops
from compactattention_amd._hip import CaError

pytestmark = pytest.mark.gpu


def _pairs(n, total, seed):
    perm = np.random.default_rng(seed).permutation(total)
    return perm[:n], perm[n:2 * n]


@pytest.mark.parametrize("n", [0, 1, 2, 447, 448, 449, 1000, 1791, 1792, 2500])
def test_copy_pages(gpu, n):
    """Several pools of different pages in one call; all other pages stay."""
    print(f"case: copy_pages n={n}", flush=True)
    total = 2 * n + 7
    g = torch.Generator().manual_seed(n)
    pools = [torch.randint(0, 256, (total, 4352), generator=g, dtype=torch.uint8),
             torch.randint(-2 ** 15, 2 ** 15, (total, 64, 128), generator=g, dtype=torch.int16).view(torch.bfloat16),
             torch.randn((total + 5, 128), generator=g), torch.randint(0, 256, (total, 16), generator=g, dtype=torch.uint8)]
    src, dst = _pairs(n, total, n)
    want = [p.clone() for p in pools]
    for p in want:
        p[torch.as_tensor(dst)] = p[torch.as_tensor(src)]
    dev = [p.to(gpu) for p in pools]
    ops.copy_pages(dev, src.tolist() if n < 400 else src, torch.as_tensor(dst, dtype=torch.int32))
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu().view(torch.uint8), w.view(torch.uint8))


def test_copy_pages_of_a_strided_pool_and_from_a_graph(gpu):
    print("case: copy_pages strided, graph", flush=True)
    records = torch.randint(0, 256, (40, 4352 + 48), dtype=torch.uint8, device=gpu)
    pool = records[:, 16:16 + 4352]
    want = records.clone()
    want[5, 16:16 + 4352], want[39, 16:16 + 4352] = want[7, 16:16 + 4352].clone(), want[0, 16:16 + 4352].clone()
    ops.copy_pages(pool, [7, 0], [5, 39])
    assert torch.equal(records, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages([pool], np.arange(10), np.arange(10, 20))  # the ids live in the graph
    big = torch.randint(0, 256, (5000, 16), dtype=torch.uint8, device=gpu)
    many = torch.cuda.CUDAGraph()
    with torch.cuda.graph(many):
        ops.copy_pages([big], np.arange(2500), np.arange(2500, 5000))
    for _ in range(3):
        big[:2500] = torch.randint(0, 256, (2500, 16), dtype=torch.uint8, device=gpu)
        many.replay()
        ops.copy_pages([big[:, :16].clone()], np.arange(2400), np.arange(2500, 4900))  # its ids take the pinned memory's place
        torch.cuda.synchronize()
        assert torch.equal(big[2500:], big[:2500])
    for _ in range(3):
        pool[:10] = torch.randint(0, 256, (10, 4352), dtype=torch.uint8, device=gpu)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool[10:20], pool[:10])


def test_copy_pages_passes_over_ids_outside_the_pools(gpu):
    """Ids in device memory that do not name a page of every pool are bounds-checked by the kernel."""
    print("case: copy_pages, ids in device memory", flush=True)
    n, total = 1000, 2100
    pools = [torch.randint(0, 256, (total + i, 48), dtype=torch.uint8, device=gpu) for i in (0, 9)]
    src, dst = (np.ascontiguousarray(x, np.int32) for x in _pairs(n, total, 3))
    want = [p.clone() for p in pools]
    ids = np.stack([src, dst])
    ids[0, 5], ids[0, 6], ids[1, 900], ids[1, 901], ids[0, 999] = -1, total, total + 3, -2 ** 31, 2 ** 31 - 1
    kept = np.array([i for i in range(n) if i not in (5, 6, 900, 901, 999)])
    for p in want:
        p[torch.as_tensor(dst[kept], device=gpu, dtype=torch.long)] = p[torch.as_tensor(src[kept], device=gpu, dtype=torch.long)]
    descs = (_hip.PagePool * 2)(*(_hip.PagePool(p.data_ptr(), 48, 48, p.shape[0]) for p in pools))
    dev = torch.from_numpy(ids).to(gpu)
    _hip.check(_hip.lib().ca_copy_pages(descs, 2, src.ctypes.data, dst.ctypes.data, n, dev.data_ptr(), ops._stream()))
    for got, w in zip(pools, want):
        assert torch.equal(got, w)


def test_copy_pages_past_32_bits(gpu):
    print("case: copy_pages in a pool of 4.5 GB", flush=True)
    total = (1 << 32) // 4352 + 60_000
    pool = torch.zeros((total, 4352), dtype=torch.uint8, device=gpu)
    x = torch.randint(0, 256, (2, 4352), dtype=torch.uint8, device=gpu)
    pool[3], pool[total - 2] = x[0], x[1]
    ops.copy_pages([pool], [3, total - 2], [total - 1, 9])
    assert torch.equal(pool[total - 1], x[0]) and torch.equal(pool[9], x[1])
    assert not pool[total - 3].any() and not pool[8].any()


@pytest.mark.parametrize("src,dst", [([0, 1], [2, 2]), ([0, 1], [1, 3]), ([4], [4]), ([0], [10]), ([10], [0])])
def test_copy_pages_refuses(gpu, src, dst):
    """A page written twice, read and written, or outside a pool: nothing is copied."""
    a, b = torch.arange(160, device=gpu, dtype=torch.int32).view(10, 16), torch.ones((12, 4), device=gpu)
    before = a.clone()
    with pytest.raises(CaError):
        ops.copy_pages([a, b], src, dst)
    assert torch.equal(a, before)


def test_copy_pages_refuses_arguments(gpu):
    a = torch.zeros((10, 16), device=gpu)
    with pytest.raises(ValueError, match="host"):
        ops.copy_pages([a], torch.tensor([0], device=gpu), [1])
    with pytest.raises(ValueError, match="destinations"):
        ops.copy_pages([a], [0, 1], [2])
    with pytest.raises(ValueError, match="integers"):
        ops.copy_pages([a], [0.5], [2])
    with pytest.raises(ValueError, match="outside"):
        ops.copy_pages([a], [-1], [2])
    with pytest.raises(ValueError, match="outside"):
        ops.copy_pages([a], [1 << 32], [2])
    with pytest.raises(ValueError, match="contiguous pages"):
        ops.copy_pages([torch.zeros((10, 16, 4), device=gpu).transpose(1, 2)], [0], [2])
    with pytest.raises(ValueError, match="pools"):
        ops.copy_pages([], [0], [2])
    with pytest.raises(ValueError, match="GPU"):
        ops.copy_pages([torch.zeros(10, 16)], [0], [2])
    with pytest.raises(CaError, match="multiples of 16"):
        ops.copy_pages([torch.zeros((10, 3), device=gpu)], [0], [2])
    with pytest.raises(CaError):
        ops.copy_pages([torch.zeros((1, 16), device=gpu).expand(10, 16)], [0], [2])
    with pytest.raises(ValueError, match="one device"):
        ops.norm_rope_qk(*(torch.zeros((1, 1, 1, 128), dtype=torch.bfloat16, device=gpu),) * 2,
                         *(torch.zeros(128, dtype=torch.bfloat16, device=gpu),) * 2, 1e-5,
                         *(_Elsewhere(torch.zeros((1, 128), device=gpu)),) * 2)


class _Elsewhere(torch.Tensor):
    """A tensor that says it is on the next GPU (there is one here)."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    def get_device(self):
        return 1


def _norm_rope64(x, w, eps, cos, sin):
    """(out, terms) in 64 bits; terms = |a cos| + |b sin| of each element, what fp32 roundings are relative to."""
    x = x.double()
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    r = torch.cat([-y[..., 64:], y[..., :64]], -1)
    return y * c + r * s, (y * c).abs() + (r * s).abs()


@pytest.mark.parametrize("B,L,Hq,Hkv,per_request,strided", [
    (1, 1, 1, 1, False, False), (1, 1, 32, 8, False, True), (8, 1, 32, 8, True, True), (2, 33, 28, 4, False, True),
    (3, 7, 9, 7, True, False), (1, 130, 24, 6, False, True), (1, 2048, 32, 8, False, True), (5, 64, 16, 1, True, True),
])
def test_norm_rope(gpu, B, L, Hq, Hkv, per_request, strided):
    print(f"case: norm_rope B={B} L={L} heads={Hq}/{Hkv} per_request={per_request} strided={strided}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(L)
    qkv = torch.randn((B, L, Hq + 2 * Hkv, 128), generator=g, device=gpu)
    qkv[:, :, ::3] *= 1000.0
    qkv[:, :, 1::5] *= 1e-4
    qkv[:, -1, 0] = 0.0  # a head of zeros: zeros
    qkv = qkv.to(torch.bfloat16)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    qw, kw = (torch.randn(128, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2))
    ang = torch.rand(((B, L, 128) if per_request else (L, 128)), generator=g, device=gpu) * 6.3
    cos, sin = ang.cos(), ang.sin()  # both halves of a row of their own
    got = ops.norm_rope_qk(q, k, qw, kw, 1e-5, cos, sin)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want, terms = _norm_rope64(x, w, 1e-5, cos, sin)
        assert y.shape == x.shape and y.is_contiguous() and y.dtype == torch.bfloat16
        # fp32: 130 roundings in the mean, halved by the root, then 8 more, 2^-24 each; the result once to bf16
        tol = 1.01 * (75 * 2.0 ** -24 * terms + 2.0 ** -8 * want.abs()) + 2.0 ** -126
        assert ((y.double() - want).abs() <= tol).all(), float(((y.double() - want).abs() / tol).max())


def test_norm_rope_of_no_tokens_and_from_a_graph(gpu):
    print("case: norm_rope empty, graph", flush=True)
    w = torch.ones(128, dtype=torch.bfloat16, device=gpu)
    e = torch.zeros((2, 0, 4, 128), dtype=torch.bfloat16, device=gpu)
    t = torch.zeros((0, 128), device=gpu)
    a, b = ops.norm_rope_qk(e, e[:, :, :1], w, w, 1e-5, t, t)
    assert a.shape == e.shape and b.shape == (2, 0, 1, 128)
    q, k = (torch.randn((2, 5, h, 128), device=gpu).to(torch.bfloat16) for h in (6, 2))
    cos, sin = torch.randn((2, 5, 128), device=gpu)
    graph = torch.cuda.CUDAGraph()
    ops.norm_rope_qk(q, k, w, w, 1e-5, cos, sin)
    with torch.cuda.graph(graph):
        held = ops.norm_rope_qk(q, k, w, w, 1e-5, cos, sin)
    for _ in range(3):
        q.normal_()
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = ops.norm_rope_qk(q, k, w, w, 1e-5, cos, sin)
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_norm_rope_nan_stays_in_its_head(gpu):
    print("case: norm_rope nan", flush=True)
    q = torch.randn((1, 3, 9, 128), device=gpu).to(torch.bfloat16)
    k = torch.randn((1, 3, 2, 128), device=gpu).to(torch.bfloat16)
    q[0, 1, 4, 100] = float("nan")
    k[0, 2, 1, 3] = float("inf")
    w = torch.ones(128, dtype=torch.bfloat16, device=gpu)
    cos, sin = torch.ones((3, 128), device=gpu), torch.zeros((3, 128), device=gpu)
    a, b = ops.norm_rope_qk(q, k, w, w, 1e-5, cos, sin)
    bad = torch.isnan(a).any(-1)
    assert bad[0, 1, 4] and bad.sum() == 1 and torch.isnan(a[0, 1, 4]).all()
    assert torch.isnan(b[0, 2, 1]).any() and torch.isfinite(b[0, :2]).all() and torch.isfinite(b[0, 2, 0]).all()
