"""The operators of a bounded KV cache, as they are timed: attention with a sliding window and sink tokens, the attention
weight that every cached key has received, and eviction of the tokens that received least.

``own`` False computes them in their plain form (elementary torch operations in fp32), True calls the package.

Query t of a request stands at position p = start + t.  Under a window it sees key j where j <= p, and p - j < window or
j < sinks.  A key's weight is summed over the queries and the heads of its KV group, exp(q . k * scale - lse).  Of a row's
tokens the first ``sinks``, the last ``recent`` and, up to ``budget`` in all, the heaviest of the others stay, in order.

Caches in 4 bits: a page holds 64 tokens of one KV head's K or V in 4352 bytes, 4096 bytes of E2M1 codes (0, 0.5, 1, 1.5,
2, 3, 4, 6 and a sign) and 256 scale bytes, one 2^(byte - 127) for every 32 head dims of a token.  K codes lie token by
token; V codes are interleaved by four tokens (token t, dims 8 m .. 8 m + 7 at byte 256 (t / 4) + 16 m + 4 (t % 4)).
Scale bytes follow at 4096: K's of token t, group g at 64 g + 4 (t % 16) + t / 16, V's at 64 g + 16 (t % 16 / 4) +
4 (t / 16) + t % 4.
"""
import math

import torch

own = False

D = 128
BLOCK = 64
PAGE = 4352
SCALE = 1.0 / math.sqrt(D)
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of one long chat, and of a ragged batch
        dict(name="window 1024, one token at 131071", op="window", starts="131071", length=1, hq=32, hkv=8, window=1024, sinks=4, kv="paged"),
        dict(name="window 4096, 16 ragged tokens", op="window", starts=",".join(str(2477 * i + 63) for i in range(16)), length=1,
             hq=32, hkv=8, window=4096, sinks=64, kv="paged"),
        # the same over pages of 4 bits, a wide window
        dict(name="window 16384, 8 tokens, 4 bits", op="window", starts=",".join(str(9001 * i + 20000) for i in range(8)), length=1,
             hq=28, hkv=4, window=16384, sinks=16, kv="q4"),
        # a prompt's chunk, and an odd one over a contiguous cache
        dict(name="window 4096, chunk of 2048", op="window", starts="30720", length=2048, hq=32, hkv=8, window=4096, sinks=64, kv="paged"),
        dict(name="window 1500, chunk of 1000", op="window", starts="9037", length=1000, hq=28, hkv=4, window=1500, sinks=5, kv="heads"),
        dict(name="window 2048, chunk of 512, 4 bits", op="window", starts="30720,6000", length=512, hq=32, hkv=8, window=2048, sinks=64,
             kv="q4"),
        # a decode step's weights
        dict(name="weights of one token, 131072", op="mass", starts="131071", length=1, hq=32, hkv=8, kv="paged", keep=1.0),
        # the last tokens of a prompt vote for the keys that a bounded cache keeps
        dict(name="weights of 64 tokens, 32768", op="mass", starts="32704", length=64, hq=32, hkv=8, kv="paged", keep=1.0),
        # every query of a chunk over the blocks that its selection kept
        dict(name="weights of a chunk, 20 % kept", op="mass", starts="30720", length=2048, hq=32, hkv=8, kv="paged", keep=0.2),
        # after a long prompt; a decode step's refill of a batch; 4-bit pages
        dict(name="evict 131072 to 8192", op="evict", lens="131072", hkv=8, budget=8192, sinks=4, recent=1024, kv="paged"),
        dict(name="evict 16 of 4160 to 4096", op="evict", lens=",".join(["4160"] * 16), hkv=8, budget=4096, sinks=4, recent=2048, kv="paged"),
        dict(name="evict ragged to 2000, 4 bits", op="evict", lens="33001,700,12345,5000", hkv=4, budget=2000, sinks=5, recent=501, kv="q4"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "window", "mass", "mass", "evict", "evict"])
    hq, hkv = rng.choice([(32, 8), (28, 4), (8, 8), (16, 2), (24, 6)])
    kv = rng.choice(["paged", "paged", "heads", "q4"])
    batch = rng.choice([1, 1, 2, 5, 16])
    if op == "evict":
        budget = _log(rng, 64, 8192 // min(batch, 8))
        sinks, recent = rng.randrange(0, 33), rng.randrange(0, budget // 2)
        lens = [_log(rng, max(16, budget // 2), 131072 // batch) for _ in range(batch)]
        return dict(op=op, lens=",".join(map(str, lens)), hkv=hkv, budget=max(budget, sinks + recent), sinks=sinks, recent=recent, kv=kv)
    length = rng.choice([1, 1, 1, 2, 3, 16, _log(rng, 32, 2048), _log(rng, 32, 2048)])
    batch = min(batch, max(1, 2048 // length)) if length > 16 else batch
    starts = [_log(rng, 16, 131072 // batch) - 16 for _ in range(batch)]
    if op == "window":
        window = _log(rng, 16, 16384 if length <= 16 else 4096)
        return dict(op=op, starts=",".join(map(str, starts)), length=length, hq=hq, hkv=hkv, window=window,
                    sinks=rng.choice([0, 1, 4, 16, 64, 200]), kv=kv)
    starts = [min(s, 32768) if length > 64 else s for s in starts]
    return dict(op=op, starts=",".join(map(str, starts)), length=length, hq=hq, hkv=hkv, kv=kv,
                keep=rng.choice([0.1, 0.2]) if length > 64 else rng.choice([0.3, 1.0, 1.0]))


def _ints(text):
    return [int(x) for x in text.split(",")]


# ----------------------------------------------------------------------------- the 4-bit format, plain
def _of_pages(pages, values):
    """Pages uint8 [n, 4352] -> fp32 values [n, 64, 128]."""
    n = pages.shape[0]
    data, scales = pages[:, :4096], pages[:, 4096:]
    if values:
        packed = data.reshape(n, 16, 16, 4, 4).transpose(2, 3).reshape(n, 64, 64)
        byte = scales.reshape(n, 4, 4, 4, 4).permute(0, 3, 2, 4, 1).reshape(n, 64, 4)
    else:
        packed = data.reshape(n, 64, 64)
        byte = scales.reshape(n, 4, 16, 4).permute(0, 3, 2, 1).reshape(n, 64, 4)
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(n, 64, D)
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=pages.device)
    scale = torch.exp2(byte.to(torch.float32) - 127.0)
    return (level[code.to(torch.int64)].view(n, 64, 4, 32) * scale[..., None]).view(n, 64, D)


def _random_pages(n, g, dev):
    """Pages of 4 bits as quantised normal values leave them: codes of a normal variable, scales about 2^-1."""
    x = torch.randn((n, 4096, 2), generator=g, device=dev) * 2.2
    a = x.abs()
    code = sum((a > edge).to(torch.uint8) for edge in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)) | ((x < 0).to(torch.uint8) << 3)
    pages = torch.empty((n, PAGE), dtype=torch.uint8, device=dev)
    pages[:, :4096] = code[..., 0] | (code[..., 1] << 4)
    pages[:, 4096:] = torch.randint(125, 128, (n, 256), generator=g, device=dev, dtype=torch.uint8)
    return pages


# ----------------------------------------------------------------------------- inputs
def _blocks(n):
    return -(-n // BLOCK)


def _seen_blocks(start, length, window, sinks):
    """The blocks that some query of a request sees under a window: (sink blocks, first block of the window, end)."""
    end = _blocks(start + length)
    first = max(0, start - window + 1) // BLOCK
    return min(_blocks(sinks), first), first, end


def _cache(kv, rows_of, batch, hkv, cap, g, dev):
    """K and V of every row: (K store, V store, page table or None).  Paged: a page for each block of rows_of[b], in no
    order, -1 for the others (blocks that a bounded cache has given back)."""
    if kv == "heads":
        return tuple(torch.randn((batch, hkv, cap * BLOCK, D), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2)) + (None,)
    table = torch.full((batch, hkv, cap), -1, dtype=torch.int32, device=dev)
    total = hkv * sum(len(r) for r in rows_of)
    perm = torch.randperm(total + 3, generator=g, device=dev)[:total].to(torch.int32)
    at = 0
    for b, r in enumerate(rows_of):
        n = hkv * len(r)
        table[b][:, torch.tensor(r, device=dev)] = perm[at:at + n].view(hkv, len(r))
        at += n
    pools = []
    for _ in range(2):
        if kv == "q4":
            pools.append(torch.cat([_random_pages(min(4096, total + 3 - i), g, dev) for i in range(0, total + 3, 4096)]))
        else:
            pools.append(torch.randn((total + 3, BLOCK, D), generator=g, device=dev, dtype=torch.bfloat16))
    return pools[0], pools[1], table.view(batch * hkv, cap)


def _tokens(st, store, values, b, h, ids):
    """fp32 [n * 64, 128]: the tokens of blocks ids (a tensor) of row (b, h)."""
    if st["table"] is None:
        return store[b, h].view(-1, BLOCK, D)[ids].reshape(-1, D).float()
    pages = store[st["table"][b * st["hkv"] + h, ids].to(torch.int64)]
    return (_of_pages(pages, values) if st["kv"] == "q4" else pages.float()).reshape(-1, D)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    op, hkv, kv = case["op"], case["hkv"], case["kv"]
    st = dict(op=op, case=case, hkv=hkv, kv=kv)
    if op == "evict":
        lens = _ints(case["lens"])
        B, budget = len(lens), case["budget"]
        cap, n = _blocks(max(lens)), _blocks(budget)
        st["k"], st["v"], st["table"] = _cache(kv, [range(_blocks(x)) for x in lens], B, hkv, cap, g, dev)
        # weights as attention leaves them: a few tokens hold most, many next to nothing or none
        w = torch.exp(3.0 * torch.randn((B * hkv, cap * BLOCK), generator=g, device=dev) - 6.0)
        st["mass"] = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.02, torch.zeros_like(w), w)
        # the pages that take what stays
        if kv == "heads":
            st["k2"], st["v2"] = (torch.zeros((B, hkv, n * BLOCK, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
            st["table2"] = None
        else:
            shape, dtype = ((PAGE,), torch.uint8) if kv == "q4" else ((BLOCK, D), torch.bfloat16)
            st["k2"], st["v2"] = (torch.zeros((B * hkv * n, *shape), dtype=dtype, device=dev) for _ in range(2))
            st["table2"] = torch.randperm(B * hkv * n, generator=g, device=dev).to(torch.int32).view(B * hkv, n)
        st["lens"] = lens
        return st
    starts, L, hq = _ints(case["starts"]), case["length"], case["hq"]
    B = len(starts)
    cap = _blocks(max(starts) + L)
    st["starts"], st["cap"] = starts, cap
    if op == "window":
        rows_of = []
        for s in starts:
            a, first, end = _seen_blocks(s, L, case["window"], case["sinks"])
            rows_of.append(list(range(a)) + list(range(first, end)))
    else:
        rows_of = [range(_blocks(s + L)) for s in starts]
    st["k"], st["v"], st["table"] = _cache(kv, rows_of, B, hkv, cap, g, dev)
    # q as the fused projection leaves it (strided)
    st["q"] = torch.randn((B, L, (hq + 2 * hkv) * D), generator=g, device=dev).to(torch.bfloat16)[..., :hq * D].view(B, L, hq, D)
    if op == "mass":
        st["v"] = None
        st["mass"] = torch.exp(3.0 * torch.randn((B * hkv, cap * BLOCK), generator=g, device=dev) - 6.0)
        st["out"] = torch.zeros_like(st["mass"])
        st["blocks"] = st["counts"] = None
        if case["keep"] < 1.0:  # every row's own blocks, in order, and the queries' own
            col = torch.arange(cap, device=dev)
            keep = torch.rand((B * hkv, cap), generator=g, device=dev) < case["keep"]
            first = torch.tensor([s // BLOCK for s in starts], device=dev).repeat_interleave(hkv)[:, None]
            end = torch.tensor([_blocks(s + L) for s in starts], device=dev).repeat_interleave(hkv)[:, None]
            keep = (keep | (col >= first)) & (col < end)
            order = torch.sort(torch.where(keep, col, col + cap), dim=1).values
            st["counts"] = keep.sum(1).to(torch.int32)
            st["blocks"] = torch.where(order < cap, order, torch.zeros_like(order)).to(torch.int32).contiguous()
        # the log-sum-exp that attention over the same keys returns
        st["lse"] = torch.empty((B, hq, L), device=dev)
        G = hq // hkv
        for b in range(B):
            for h in range(hkv):
                s, _ = _scores(st, b, h)
                st["lse"][b, h * G:(h + 1) * G] = torch.logsumexp(s, -1).view(L, G).t()
    return st


# ----------------------------------------------------------------------------- one pass
def _listed_blocks(st, b, h):
    dev = st["q"].device
    if st.get("blocks") is None:
        return torch.arange(_blocks(st["starts"][b] + st["q"].shape[1]), device=dev)
    r = b * st["hkv"] + h
    return st["blocks"][r, :int(st["counts"][r])].to(torch.int64)


def _scores(st, b, h):
    """fp32 scores [L * G, keys] of row (b, h) over its listed blocks, hidden ones -inf, and the keys' positions."""
    q, start = st["q"], st["starts"][b]
    _, L, Hq, _ = q.shape
    G = Hq // st["hkv"]
    ids = _listed_blocks(st, b, h)
    K = _tokens(st, st["k"], False, b, h, ids)
    kpos = (ids[:, None] * BLOCK + torch.arange(BLOCK, device=q.device)).reshape(-1)
    s = torch.matmul(q[b, :, h * G:(h + 1) * G].float().reshape(L * G, D), K.t()) * SCALE
    qpos = (start + torch.arange(L, device=q.device)).repeat_interleave(G)
    return s.masked_fill_(kpos[None, :] > qpos[:, None], float("-inf")), kpos


def _window(st):
    q, case = st["q"], st["case"]
    B, L, Hq, _ = q.shape
    H = st["hkv"]
    G = Hq // H
    dev = q.device
    W, S = case["window"], case["sinks"]
    out = torch.empty((B, L, Hq, D), dtype=torch.bfloat16, device=dev)
    for b in range(B):
        start = st["starts"][b]
        a, first, end = _seen_blocks(start, L, W, S)
        ids = torch.cat([torch.arange(a, device=dev), torch.arange(first, end, device=dev)])
        n = ids.numel()
        if st["table"] is None:
            K, V = (x[b].view(H, -1, BLOCK, D)[:, ids].reshape(H, n * BLOCK, D).float() for x in (st["k"], st["v"]))
        else:
            pages = st["table"].view(B, H, -1)[b][:, ids].reshape(-1).to(torch.int64)
            if st["kv"] == "q4":
                K, V = (_of_pages(x[pages], i == 1).view(H, n * BLOCK, D) for i, x in enumerate((st["k"], st["v"])))
            else:
                K, V = (x[pages].view(H, n * BLOCK, D).float() for x in (st["k"], st["v"]))
        kpos = (ids[:, None] * BLOCK + torch.arange(BLOCK, device=dev)).reshape(-1)
        qpos = (start + torch.arange(L, device=dev)).repeat_interleave(G)[:, None]
        seen = (kpos <= qpos) & ((qpos - kpos < W) | (kpos < S))
        qr = q[b].float().view(L, H, G, D).transpose(0, 1).reshape(H, L * G, D)
        s = torch.matmul(qr, K.transpose(1, 2).contiguous()) * SCALE
        s = s.masked_fill_(~seen, float("-inf"))
        s = s - s.amax(-1, keepdim=True)
        p = torch.exp(s)
        o = torch.matmul(p, V) / p.sum(-1, keepdim=True)
        out[b] = o.view(H, L, G, D).transpose(0, 1).reshape(L, Hq, D).to(torch.bfloat16)
    return out


def _mass(st):
    q, out = st["q"], st["out"]
    B, L, Hq, _ = q.shape
    H = st["hkv"]
    G = Hq // H
    for b in range(B):
        end = st["starts"][b] + L
        out[b * H:(b + 1) * H, :end] = st["mass"][b * H:(b + 1) * H, :end]
        for h in range(H):
            s, kpos = _scores(st, b, h)
            lse = st["lse"][b, h * G:(h + 1) * G].t().reshape(L * G, 1)
            w = torch.exp(s - lse).sum(0)
            there = kpos < end
            out[b * H + h].index_add_(0, kpos[there], w[there])
    return out


def _evict(st):
    case, lens, H = st["case"], st["lens"], st["hkv"]
    B, budget, S, R = len(lens), case["budget"], case["sinks"], case["recent"]
    dev = st["mass"].device
    keep = torch.full((B * H, budget), -1, dtype=torch.int32, device=dev)
    moved = torch.zeros((B * H, budget), device=dev)
    q4 = st["kv"] == "q4"
    back = [torch.zeros((B, H, budget, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    for b, n in enumerate(lens):
        for h in range(H):
            r = b * H + h
            if n <= budget:
                ids = torch.arange(n, device=dev)
            else:
                m = st["mass"][r, :n].clone()
                m[:S] = float("inf")
                m[n - R:] = float("inf")
                ids = torch.sort(torch.sort(m, descending=True, stable=True).indices[:budget]).values
            k = ids.numel()
            keep[r, :k] = ids.to(torch.int32)
            moved[r, :k] = st["mass"][r, ids]
            for src, dst, tokens, values in ((st["k"], st["k2"], back[0], False), (st["v"], st["v2"], back[1], True)):
                if q4:  # the bytes of every token, to their places in other pages
                    sp, st_ = st["table"][r, ids // BLOCK].to(torch.int64), ids % BLOCK
                    j = torch.arange(k, device=dev)
                    dp, dt = st["table2"][r, j // BLOCK].to(torch.int64), j % BLOCK
                    flat = dst.view(-1)
                    flat[dp[:, None] * PAGE + _token_bytes(dt, values)] = src.view(-1)[sp[:, None] * PAGE + _token_bytes(st_, values)]
                    x = _of_pages(dst[st["table2"][r, :_blocks(k)].to(torch.int64)], values).reshape(-1, D)[:k]
                    tokens[b, h, :k] = x.to(torch.bfloat16)
                    continue
                if st["table"] is None:
                    dst[b, h, :k] = src[b, h, ids]
                    tokens[b, h, :k] = dst[b, h, :k]
                    continue
                x = src[st["table"][r, ids // BLOCK].to(torch.int64), ids % BLOCK]
                j = torch.arange(k, device=dev)
                dst[st["table2"][r, j // BLOCK].to(torch.int64), j % BLOCK] = x
    if q4:
        return keep, moved, back[0], back[1]
    return keep, moved, st["k2"], st["v2"]


def _token_bytes(t, values):
    """The places of a token's 68 bytes in its page, [n, 68]."""
    i = torch.arange(64, device=t.device)
    grp = torch.arange(4, device=t.device)
    t = t[:, None]
    if values:
        return torch.cat([256 * (t // 4) + 16 * (i // 4) + 4 * (t % 4) + i % 4,
                          4096 + 64 * grp + 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4], 1)
    return torch.cat([64 * t + i, 4096 + 64 * grp + 4 * (t % 16) + t // 16], 1)


def _layout(ops, st, store, table):
    if table is None:
        return ops.KV.heads_first(store)
    return ops.KV4.paged(store, table) if st["kv"] == "q4" else ops.KV.paged(store, table)


def run(st):
    op, case, H = st["op"], st["case"], st["hkv"]
    if not own:
        return {"window": _window, "mass": _mass, "evict": _evict}[op](st)
    from compactattention_amd import ops

    K = _layout(ops, st, st["k"], st["table"])
    if op == "window":
        V = _layout(ops, st, st["v"], st["table"])
        return ops.attn_window(st["q"], K, V, st["starts"], case["window"], case["sinks"], SCALE, st["cap"], H)
    if op == "mass":
        return ops.key_mass(st["q"], K, st["lse"], st["mass"], st["starts"], SCALE, st["cap"], H, table=st["blocks"],
                            counts=st["counts"], out=st["out"])
    lens, budget = st["lens"], case["budget"]
    V = _layout(ops, st, st["v"], st["table"])
    K2, V2 = _layout(ops, st, st["k2"], st["table2"]), _layout(ops, st, st["v2"], st["table2"])
    keep = ops.heavy_tokens(st["mass"], lens, H, budget, case["sinks"], case["recent"])
    moved = ops.move_tokens(K, V, K2, V2, keep, lens, H, mass=st["mass"])
    if st["kv"] != "q4":
        return keep, moved, st["k2"], st["v2"]
    return keep, moved, *ops.gather_q4(K2, V2, len(lens), H, 0, budget)  # what the pages now stand for


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, hkv = case["op"], case["hkv"]
    token = 68 if case["kv"] == "q4" else 2 * D  # of K, or of V
    if op == "evict":
        n = m = 0
        for x in _ints(case["lens"]):
            n += hkv * min(x, case["budget"])
            m += hkv * x
        back = 2 * 2 * D * n if case["kv"] == "q4" else 0  # the values that the pages stand for
        return {"bytes": 4 * m + n * (2 * 2 * token + 4 + 4) + back, "flops": 0}
    starts, L, hq = _ints(case["starts"]), case["length"], case["hq"]
    keys = pairs = 0
    for s in starts:
        if op == "window":
            W, S = case["window"], case["sinks"]
            lo = max(0, s - W + 1)
            keys += hkv * (s + L - lo + min(S, lo))
            for t in range(L):
                p = s + t
                first = max(0, p - W + 1)
                pairs += hq * (p + 1 - first + min(S, first))
        else:
            kept = case["keep"] * s
            keys += hkv * (kept + L)
            pairs += hq * (L * kept + L * (L + 1) / 2)
    q = len(starts) * L * hq
    if op == "window":
        return {"bytes": keys * 2 * token + 2 * q * 2 * D, "flops": 4 * D * pairs}
    tokens = hkv * sum(s + L for s in starts)  # their weights, read and written
    return {"bytes": keys * token + q * (2 * D + 4) + 8 * tokens, "flops": 2 * D * pairs}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _level64(code):
    """The value of E2M1 codes: sign, two exponent bits, one mantissa bit."""
    s = 1.0 - 2.0 * (code >> 3).double()
    e, m = ((code >> 1) & 3).double(), (code & 1).double()
    return s * torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)


def _row64(st, store, table, values, b, h, tokens):
    """fp64 [n, 128]: tokens (positions, a tensor) of row (b, h), each element looked up at its own place."""
    blk, t = tokens // BLOCK, tokens % BLOCK
    if table is None:
        return store[b, h, tokens].double()
    page = table[b * st["hkv"] + h, blk].to(torch.int64)
    if st["kv"] != "q4":
        return store[page, t].double()
    d = torch.arange(D, device=tokens.device)[None, :]
    g, t = d // 32, t[:, None]
    if values:
        at, sat = 256 * (t // 4) + 16 * (d // 8) + 4 * (t % 4) + d % 8 // 2, 64 * g + 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4
    else:
        at, sat = 64 * t + d // 2, 64 * g + 4 * (t % 16) + t // 16
    flat = store.view(-1)
    byte = flat[page[:, None] * PAGE + at].to(torch.int32)
    code = torch.where(d % 2 == 1, byte >> 4, byte & 15)
    return _level64(code) * torch.exp2(flat[page[:, None] * PAGE + 4096 + sat].double() - 127)


def exact(case, seed):
    st = prepare(case, seed)
    op, H = case["op"], case["hkv"]
    if op == "evict":
        lens, budget, S, R = st["lens"], case["budget"], case["sinks"], case["recent"]
        dev = st["mass"].device
        B = len(lens)
        keep = torch.full((B * H, budget), -1, dtype=torch.int32, device=dev)
        moved = torch.zeros((B * H, budget), dtype=torch.float64, device=dev)
        k2, v2 = (torch.zeros((B, H, _blocks(budget) * BLOCK, D), dtype=torch.float64, device=dev) for _ in range(2))
        for b, n in enumerate(lens):
            for h in range(H):
                m = st["mass"][b * H + h, :n].double()
                fixed = [j for j in range(n) if n <= budget or j < S or j >= n - R]
                middle = m[S:n - R].cpu().tolist() if n > budget else []
                order = sorted(range(len(middle)), key=lambda j: (-middle[j], j))[:budget - S - R]
                ids = torch.tensor(sorted(fixed + [S + j for j in order]), device=dev)
                keep[b * H + h, :ids.numel()] = ids.to(torch.int32)
                moved[b * H + h, :ids.numel()] = m[ids]
                k2[b, h, :ids.numel()] = _row64(st, st["k"], st["table"], False, b, h, ids)
                v2[b, h, :ids.numel()] = _row64(st, st["v"], st["table"], True, b, h, ids)
        if case["kv"] == "q4":
            return keep, moved, k2[:, :, :budget], v2[:, :, :budget]
        if case["kv"] == "paged":  # by page
            outs = []
            for x in (k2, v2):
                pool = torch.empty((st["k2"].shape[0], BLOCK, D), dtype=torch.float64, device=dev)
                pool[st["table2"].reshape(-1).to(torch.int64)] = x.view(-1, BLOCK, D)
                outs.append(pool)
            return keep, moved, outs[0], outs[1]
        return keep, moved, k2, v2
    q = st["q"]
    B, L, Hq, _ = q.shape
    G = Hq // H
    dev = q.device
    if op == "mass":
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device=dev)
        for b in range(B):
            for h in range(H):
                r = b * H + h
                n = st["starts"][b] + L
                out[r, :n] = st["mass"][r, :n].double()
                pos = torch.arange(n, device=dev)
                if st["blocks"] is not None:
                    held = torch.zeros(st["cap"], dtype=torch.bool, device=dev)
                    held[st["blocks"][r, :int(st["counts"][r])].to(torch.int64)] = True
                    pos = pos[held[pos // BLOCK]]
                k = _row64(st, st["k"], st["table"], False, b, h, pos)
                for t0 in range(0, L, 256):
                    for gq in range(G):
                        x = q[b, t0:t0 + 256, h * G + gq].double()
                        at = st["starts"][b] + t0 + torch.arange(x.shape[0], device=dev)
                        e = torch.exp(torch.matmul(x, k.t()) / math.sqrt(D) - st["lse"][b, h * G + gq, t0:t0 + 256].double()[:, None])
                        out[r, pos] += torch.where(pos[None, :] <= at[:, None], e, torch.zeros_like(e)).sum(0)
        return out
    W, S = case["window"], case["sinks"]
    out = torch.empty((B, L, Hq, D), dtype=torch.float64, device=dev)
    for b in range(B):
        start = st["starts"][b]
        for h in range(H):
            for t0 in range(0, L, 512):
                n = min(512, L - t0)
                lo = max(0, start + t0 - W + 1)
                pos = torch.cat([torch.arange(min(S, lo), device=dev), torch.arange(lo, start + t0 + n, device=dev)])
                k, v = _row64(st, st["k"], st["table"], False, b, h, pos), _row64(st, st["v"], st["table"], True, b, h, pos)
                at = (start + t0 + torch.arange(n, device=dev))[:, None]
                hidden = (pos > at) | ((at - pos >= W) & (pos >= S))
                for gq in range(G):
                    s = torch.matmul(q[b, t0:t0 + n, h * G + gq].double(), k.t()) / math.sqrt(D)
                    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                    out[b, t0:t0 + n, h * G + gq] = torch.matmul(p, v)
    return out
