"""Window attention, the weight that keys received and eviction in 64 bits, written from their definitions, and caches to
run them on."""
from __future__ import annotations

import math

import numpy as np
import torch

from compactattention_amd import ops
from tests import kv4_oracle

D, BLOCK = 128, 64
SCALE = 1.0 / math.sqrt(D)


class Cache:
    """Keys and values [B, Hkv, N, 128] (bf16 values, fp64 on the CPU; in 4 bits what the pages stand for) and the layouts
    that the operators take.  kind: heads, seq, paged, q4.  Paged rows have pages, in no order, for the blocks of
    ``blocks`` (all of them if None); other entries are -1, and page 0, which a clamped -1 would read, is NaN."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, kind: str, device, seed: int = 0, blocks=None):
        self.kind, (self.B, self.H, self.N, _) = kind, k.shape
        self.cap = -(-self.N // BLOCK)
        self.device = torch.device(device)
        pad = torch.zeros((self.B, self.H, self.cap * BLOCK - self.N, D), dtype=torch.bfloat16)
        full = [torch.cat([t, pad], 2) for t in (k, v)]
        self.k, self.v = k.double(), v.double()
        if kind == "heads":
            self.stores = [t.to(device) for t in (k, v)]
            self.K, self.V = (ops.KV.heads_first(t) for t in self.stores)
            return
        if kind == "seq":
            self.stores = [t.transpose(1, 2).contiguous().to(device) for t in (k, v)]
            self.K, self.V = (ops.KV.seq_first(t) for t in self.stores)
            return
        used = list(range(self.cap)) if blocks is None else sorted(blocks)
        rows = self.B * self.H
        g = torch.Generator().manual_seed(seed + 1)
        self.ids = 1 + torch.randperm(rows * len(used), generator=g).view(rows, len(used))
        table = torch.full((rows, self.cap), -1, dtype=torch.int32)
        table[:, used] = self.ids.to(torch.int32)
        self.stores = []
        for i, t in enumerate(full):
            tokens = t.view(rows, self.cap, BLOCK, D)[:, used].reshape(-1, BLOCK, D)
            at = self.ids.reshape(-1)
            if kind == "q4":
                pool = torch.full((rows * len(used) + 1, kv4_oracle.PAGE), 255, dtype=torch.uint8)
                pool[at] = kv4_oracle.make_pages(tokens, i == 1)
                back = kv4_oracle.read_pages(pool[at], i == 1).view(rows, len(used) * BLOCK, D)
                held = torch.zeros((rows, self.cap * BLOCK, D), dtype=torch.float64)
                held.view(rows, self.cap, BLOCK, D)[:, used] = back.view(rows, len(used), BLOCK, D)
                setattr(self, "kv"[i], held.view(self.B, self.H, -1, D)[:, :, :self.N])
            else:
                pool = torch.full((rows * len(used) + 1, BLOCK, D), math.nan, dtype=torch.bfloat16)
                pool[at] = tokens
            self.stores.append(pool.to(device))
        self.table = table.to(device)
        make = ops.KV4.paged if kind == "q4" else ops.KV.paged
        self.K, self.V = (make(p, self.table) for p in self.stores)


def random_kv(B, H, N, seed, wide=True):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn((2, B, H, N, D), generator=g).unbind(0)
    if wide:
        k = k * (1 + 2 * (torch.rand(D, generator=g) > 0.9))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def random_q(B, L, Hq, seed, device, strided=False):
    g = torch.Generator().manual_seed(seed + 77)
    q = torch.randn((B, L, Hq + 3, D), generator=g).to(torch.bfloat16).to(device)
    return q[:, :, 1:Hq + 1] if strided else q[:, :, :Hq].contiguous()


def visible(p: int, kpos: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    """Which positions a query at p sees (window 0: all up to p)."""
    seen = kpos <= p
    return seen if window == 0 else seen & ((p - kpos < window) | (kpos < sinks))


def blocks_seen(start, L, window, sinks):
    """Blocks with a key that some query at start .. start + L - 1 sees."""
    kpos = torch.arange(start + L)
    seen = visible(start, kpos, window, sinks)
    seen[max(0, start - window + 1):] = True  # every key from the first query's window on is some query's
    return sorted(set((seen.nonzero()[:, 0] // BLOCK).tolist()))


def attention(q, cache: Cache, starts, window, sinks, scale=SCALE):
    """(out [B, L, Hq, 128], lse [B, Hq, L], tolerance of out, of lse) in 64 bits, hidden keys left out altogether."""
    q = q.cpu().double()
    B, L, Hq, _ = q.shape
    G = Hq // cache.H
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse, ltol = torch.zeros((B, Hq, L), dtype=torch.float64), torch.zeros((B, Hq, L), dtype=torch.float64)
    for b in range(B):
        kpos = torch.arange(starts[b] + L)
        for t in range(L):
            seen = visible(starts[b] + t, kpos, window, sinks).nonzero()[:, 0]
            for h in range(cache.H):
                hs = slice(h * G, (h + 1) * G)
                k, v, x = cache.k[b, h, seen], cache.v[b, h, seen], q[b, t, hs]
                s = (x @ k.t()) * scale
                w = torch.softmax(s, -1)
                out[b, t, hs] = w @ v
                lse[b, hs, t] = torch.logsumexp(s, -1)
                S = (x.abs() @ k.abs().t()).amax(-1) * scale
                tol[b, t, hs] = kv4_oracle.tolerance(out[b, t, hs], w @ v.abs(), S)
                ltol[b, hs, t] = kv4_oracle.lse_tolerance(S)
    return out, lse, tol, ltol


def weights(q, cache: Cache, lse, mass, starts, window, sinks, lists=None, scale=SCALE):
    """(mass with the weights of the queries added [B*H, N] in 64 bits, its tolerance).  lists: blocks of every row.

    A weight's argument in log2 units has the score's error, 128 products and sums in fp32 and the scale (130 roundings of
    2^-24 of sum |q k| scale log2 e), two roundings of the lse's part and one of the sum; exp2 is good to 2^-22; the
    queries' weights are added one by one over tiles of 32 rows, 5 joins of lanes, 8 of waves and one to the old value."""
    q, lse = q.cpu().double(), lse.cpu().double()
    B, L, Hq, _ = q.shape
    H = cache.H
    G = Hq // H
    out = torch.as_tensor(mass).cpu().double().clone()
    tol = torch.zeros_like(out)
    eps, log2e = 2.0 ** -24, 1.4427
    adds = L * G // 32 + 16
    for b in range(B):
        kpos = torch.arange(starts[b] + L)
        for h in range(H):
            r = b * H + h
            allowed = torch.ones_like(kpos, dtype=torch.bool)
            if lists is not None:
                allowed = torch.isin(kpos // BLOCK, torch.as_tensor(lists[r], dtype=torch.int64))
            add, err = torch.zeros(kpos.numel(), dtype=torch.float64), torch.zeros(kpos.numel(), dtype=torch.float64)
            for t in range(L):
                seen = (visible(starts[b] + t, kpos, window, sinks) & allowed).nonzero()[:, 0]
                k, x = cache.k[b, h, seen], q[b, t, h * G:(h + 1) * G]
                le = lse[b, h * G:(h + 1) * G, t]
                s = (x @ k.t()) * scale
                w = torch.exp(s - le[:, None])
                w[le == -math.inf] = 0.0
                S = (x.abs() @ k.abs().t()) * scale
                a = log2e * eps * (131 * S + 3 * torch.where(torch.isfinite(le), le.abs(), 0.0)[:, None])
                add[seen] += w.sum(0)
                err[seen] += (w * (0.7 * a + 2.0 ** -22) * 1.02).sum(0)
            n = kpos.numel()
            err += eps * adds * add
            out[r, :n] += add
            tol[r, :n] = err + 2 * eps * out[r, :n].abs() + 2.0 ** -140
    return out, tol


def kept(mass: np.ndarray, n: int, budget: int, sinks: int, recent: int) -> list:
    """The positions that stay of a row's n tokens."""
    if n <= budget:
        return list(range(n))
    fixed = [j for j in range(n) if j < sinks or j >= n - recent]
    middle = [(-math.inf if math.isnan(mass[j]) else float(mass[j]), -j, math.isnan(mass[j])) for j in range(sinks, n - recent)]
    order = sorted(range(len(middle)), key=lambda i: (middle[i][2], -middle[i][0], i))
    return sorted(fixed + [sinks + i for i in order[:budget - sinks - recent]])
