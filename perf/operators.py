"""The KV-cache operators beside the bf16 attention path, as they are timed: a cache held in 4 bits (append, read back,
attention of single tokens and of chunks), copies of cache pages, and the norm of queries and keys with their rotation.

``own`` False computes them in their plain form (elementary torch operations in fp32), True calls the package.

The 4-bit cache.  A page holds 64 tokens of one KV head's K or V in 4352 bytes: 4096 bytes of E2M1 codes (0, 0.5, 1, 1.5,
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
EPS = 1e-6
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of eight requests, the queries and keys of one layer
        dict(name="norm+rotation, 8 single tokens", op="norm_rope", batch=8, length=1, hq=32, hkv=8, start=40000),
        # a chunk's q and k as the fused projection leaves them (strided)
        dict(name="norm+rotation, chunk of 2048", op="norm_rope", batch=1, length=2048, hq=32, hkv=8, start=30720),
        # a decode step's append for sixteen requests of different lengths
        dict(name="append, 16 single tokens", op="append", starts=",".join(str(977 * i + 63) for i in range(16)), length=1, hkv=8),
        # a prompt chunk's append
        dict(name="append, chunk of 2048", op="append", starts="30720", length=2048, hkv=8),
        # decode steps: a short chat, a ragged batch, the longest context
        dict(name="decode, 4096 tokens", op="decode", lens="4096", length=1, hq=32, hkv=8),
        dict(name="decode, ragged batch", op="decode", lens="254,31001,2047,9000,16385,640,23110,4999", length=1, hq=28, hkv=4),
        dict(name="decode, 131072 tokens", op="decode", lens="131072", length=1, hq=32, hkv=8),
        # a draft of 16 tokens checked in one step (more rows than one token's)
        dict(name="decode, 16 tokens at 20011", op="decode", lens="20011", length=16, hq=32, hkv=8),
        # a chunk over the blocks that the selection keeps, and a ragged batch of short dense chunks
        dict(name="chunk of 1024 over 65536, 20 % kept", op="chunk", past="1024", length=1024, hq=32, hkv=8, keep=0.2),
        dict(name="chunks of 500, ragged, dense", op="chunk", past="16,48,96,128", length=500, hq=28, hkv=4, keep=1.0),
        # copy-on-write of the last page of every row after a fork, bf16 pages
        dict(name="copy 32 bf16 pages", op="copy", pages=32, pool=8192, bits=16),
        # compaction of a pool of 4-bit pages that is a third full
        dict(name="copy 9001 4-bit pages", op="copy", pages=9001, pool=32768, bits=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "decode", "decode", "chunk", "chunk", "copy"])
    hq, hkv = rng.choice([(32, 8), (28, 4), (8, 8), (16, 2), (24, 6)])
    if op == "norm_rope":
        batch = rng.choice([1, 2, 5, 8])
        length = _log(rng, 1, 2048 // batch)
        return dict(op=op, batch=batch, length=length, hq=hq, hkv=hkv, start=rng.randrange(0, 100000))
    if op == "append":
        batch = rng.choice([1, 1, 3, 16])
        length = _log(rng, 1, 2048 // batch)
        return dict(op=op, starts=",".join(str(rng.randrange(0, 16000)) for _ in range(batch)), length=length, hkv=hkv)
    if op == "decode":
        batch = rng.choice([1, 1, 2, 5, 8])
        length = rng.choice([1, 1, 1, 2, 3, 9, 16])
        lens = [max(length, _log(rng, 16, 131072 // batch)) for _ in range(batch)]
        return dict(op=op, lens=",".join(map(str, lens)), length=length, hq=hq, hkv=hkv)
    if op == "chunk":
        batch = rng.choice([1, 1, 2, 4])
        length = _log(rng, 32, 1024 // batch)
        past = [_log(rng, 1, 512 // batch) for _ in range(batch)]
        return dict(op=op, past=",".join(map(str, past)), length=length, hq=hq, hkv=hkv, keep=rng.choice([0.1, 0.25, 0.5, 1.0]))
    bits = rng.choice([4, 16])
    pages = _log(rng, 1, 9000 if bits == 4 else 2300)
    return dict(op=op, pages=pages, pool=rng.randrange(3 * pages + 8, 3 * pages + 1000), bits=bits)


def _ints(text):
    return [int(x) for x in text.split(",")]


# ----------------------------------------------------------------------------- the 4-bit format, plain
def _codes(x):
    """fp32 [..., 128] (bf16 values) -> (E2M1 codes uint8 [..., 128], scale bytes uint8 [..., 4])."""
    g = x.reshape(*x.shape[:-1], 4, 32)
    amax = g.abs().amax(-1)
    bits = amax.to(torch.bfloat16).view(torch.int16).to(torch.int32)
    byte = (((bits + 0x1F) >> 7) - 2).clamp(2, 252)
    bad = ~torch.isfinite(amax)
    y = g * torch.exp2((127 - byte).to(torch.float32))[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.reshape(x.shape), torch.where(bad, torch.full_like(byte, 255), byte).to(torch.uint8)


def _to_pages(code, byte, values):
    """Codes [n, 64, 128] and scale bytes [n, 64, 4] -> pages uint8 [n, 4352] (values: V's order, else K's)."""
    n = code.shape[0]
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    if values:
        data = packed.view(n, 16, 4, 16, 4).transpose(2, 3).reshape(n, 4096)
        scales = byte.view(n, 4, 4, 4, 4).permute(0, 4, 2, 1, 3).reshape(n, 256)  # [t/16, t%16/4, t%4, g] -> [g, t%16/4, t/16, t%4]
    else:
        data = packed.reshape(n, 4096)
        scales = byte.view(n, 4, 16, 4).permute(0, 3, 2, 1).reshape(n, 256)  # [t/16, t%16, g] -> [g, t%16, t/16]
    return torch.cat([data, scales], 1)


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
    val = level[code.to(torch.int64)].view(n, 64, 4, 32)
    scale = torch.exp2(byte.to(torch.float32) - 127.0)
    scale = torch.where(byte == 255, torch.full_like(scale, float("nan")), scale)
    return (val * scale[..., None]).view(n, 64, D)


def _rotate_half(x):
    return torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)


# ----------------------------------------------------------------------------- inputs
def _generator(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _states(n, g, dev, channels):
    """bf16-rounded keys or values [n, 64, 128]: a few channels are several times the others, as in real keys."""
    x = torch.randn((n, BLOCK, D), generator=g, device=dev)
    return (x * channels).to(torch.bfloat16).to(torch.float32)


def _pools(pages, g, dev):
    """K and V pools of 4-bit pages with tokens quantised in them (a thousand pages at a time, to keep memory small)."""
    wide = 1.0 + 3.0 * (torch.rand(D, generator=g, device=dev) > 0.95)
    pools = []
    for values in (False, True):
        parts = []
        for p in range(0, pages, 4096):
            code, byte = _codes(_states(min(4096, pages - p), g, dev, torch.ones_like(wide) if values else wide))
            parts.append(_to_pages(code, byte, values))
        pools.append(torch.cat(parts))
    return pools


def _table(rows, blocks, g, dev, spare=3):
    """A page table [rows, max(blocks)] int32 of pages in no order; ``blocks`` pages a row."""
    width = max(blocks)
    total = rows * width + spare
    perm = torch.randperm(total, generator=g, device=dev)[:rows * width]
    return perm.view(rows, width).to(torch.int32), total


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = _generator(seed, dev)
    op = case["op"]
    st = dict(op=op, case=case)
    if op == "norm_rope":
        B, L, hq, hkv = case["batch"], case["length"], case["hq"], case["hkv"]
        qkv = torch.randn((B, L, (hq + 2 * hkv) * D), generator=g, device=dev).to(torch.bfloat16)
        st["q"] = qkv[..., :hq * D].view(B, L, hq, D)
        st["k"] = qkv[..., hq * D:(hq + hkv) * D].view(B, L, hkv, D)
        st["qw"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
        st["kw"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
        pos = torch.arange(case["start"], case["start"] + L, dtype=torch.float64, device=dev)
        freq = 500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        ang = torch.outer(pos, freq)
        ang = torch.cat([ang, ang], -1)
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        return st
    if op == "append":
        starts, L, hkv = _ints(case["starts"]), case["length"], case["hkv"]
        B = len(starts)
        blocks = [-(-(s + L) // BLOCK) for s in starts]
        st["table"], total = _table(B * hkv, blocks, g, dev)
        st["kp"], st["vp"] = torch.zeros((2, total, PAGE), dtype=torch.uint8, device=dev).unbind(0)
        st["k"] = (2 * torch.randn((B, L, hkv, D), generator=g, device=dev)).to(torch.bfloat16)
        st["v"] = torch.randn((B, L, hkv, D), generator=g, device=dev).to(torch.bfloat16)
        st["starts"], st["cap"] = starts, max(blocks)
        return st
    if op == "copy":
        n, pool = case["pages"], case["pool"]
        if case["bits"] == 4:
            st["pools"] = [torch.randint(0, 256, (pool, PAGE), generator=g, device=dev, dtype=torch.uint8) for _ in range(2)]
        else:
            st["pools"] = [torch.randn((pool, BLOCK, D), generator=g, device=dev).to(torch.bfloat16) for _ in range(2)]
        # page ids as an allocator on the host keeps them
        perm = torch.randperm(pool, generator=g, device=dev)[:2 * n].to(torch.int32).cpu().numpy()
        st["src"], st["dst"] = perm[:n], perm[n:]
        return st
    hq, hkv, L = case["hq"], case["hkv"], case["length"]
    if op == "decode":
        lens = _ints(case["lens"])
        blocks = [-(-n // BLOCK) for n in lens]
        st["lens"] = lens
    else:
        past = _ints(case["past"])
        blocks = [p + -(-L // BLOCK) for p in past]
        st["past"] = past
    B, cap = len(blocks), max(blocks)
    st["table"], total = _table(B * hkv, blocks, g, dev)
    st["kp"], st["vp"] = _pools(total, g, dev)
    st["cap"] = cap
    st["q"] = torch.randn((B, L, hq, D), generator=g, device=dev).to(torch.bfloat16)
    if op == "chunk":
        # every row keeps its own past blocks (in order) and the chunk's
        col = torch.arange(cap, device=dev)
        pastv = torch.tensor(past, device=dev).repeat_interleave(hkv)[:, None]
        nb = torch.tensor(blocks, device=dev).repeat_interleave(hkv)[:, None]
        keep = torch.rand((B * hkv, cap), generator=g, device=dev) < case["keep"]
        keep = (keep | (col >= pastv)) & (col < nb)
        order = torch.sort(torch.where(keep, col, col + cap), dim=1).values
        st["counts"] = keep.sum(1).to(torch.int32)
        st["blocks"] = torch.where(order < cap, order, torch.zeros_like(order)).to(torch.int32).contiguous()
    return st


# ----------------------------------------------------------------------------- one pass
def _norm_rope(st):
    def one(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        return (y * st["cos"][None, :, None] + _rotate_half(y) * st["sin"][None, :, None]).to(torch.bfloat16)

    return one(st["q"], st["qw"]), one(st["k"], st["kw"])


def _append(st):
    k, starts = st["k"], st["starts"]
    B, L, H, _ = k.shape
    dev = k.device
    pos = torch.tensor(starts, device=dev)[:, None] + torch.arange(L, device=dev)  # [B, L]
    pages = torch.gather(st["table"].view(B, H, -1).to(torch.int64), 2, (pos // BLOCK)[:, None].expand(B, H, L))
    t = (pos % BLOCK)[:, None, :, None]
    m = torch.arange(16, device=dev)
    grp = torch.arange(4, device=dev)
    i4 = torch.arange(4, device=dev)
    back = []
    for new, pool, values in ((k, st["kp"], False), (st["v"], st["vp"], True)):
        code, byte = _codes(new.transpose(1, 2).float())  # [B, H, L, 128], [B, H, L, 4]
        packed = (code[..., 0::2] | (code[..., 1::2] << 4)).view(B, H, L, 16, 4)
        if values:
            at = 256 * (t // 4) + 4 * (t % 4) + 16 * m
            sat = 64 * grp + 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4
        else:
            at = 64 * t + 4 * m
            sat = 64 * grp + 4 * (t % 16) + t // 16
        at = (at[..., None] + i4).expand(B, H, L, 16, 4)
        sat = (4096 + sat).expand(B, H, L, 4)
        base = pages * PAGE
        flat = pool.view(-1)
        flat[(base[..., None, None] + at)] = packed
        flat[base[..., None] + sat] = byte
        # read back what the cache now stands for
        p = flat[base[..., None, None] + at].view(B, H, L, 64)
        c = torch.stack([p & 15, p >> 4], -1).view(B, H, L, 4, 32)
        level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=dev)
        val = level[c.to(torch.int64)] * torch.exp2(flat[base[..., None] + sat].float() - 127.0)[..., None]
        back.append(val.view(B, H, L, D).to(torch.bfloat16))
    return tuple(back)


def _attend(st):
    """Queries [B, L, Hq, 128] at positions qpos0[b] + t over the blocks of every KV row's list, fp32."""
    q, table = st["q"], st["table"]
    B, L, Hq, _ = q.shape
    rows, cap = table.shape
    H = rows // B
    G = Hq // H
    dev = q.device
    if st["op"] == "decode":
        qpos0 = torch.tensor([n - L for n in st["lens"]], device=dev)
        ids = torch.arange(cap, device=dev).expand(rows, cap)
        listed_ = torch.ones((rows, cap), dtype=torch.bool, device=dev)
    else:
        qpos0 = torch.tensor([BLOCK * p for p in st["past"]], device=dev)
        width = int(cap)
        ids = st["blocks"][:, :width].to(torch.int64)
        listed_ = torch.arange(width, device=dev) < st["counts"][:, None]
        used = max(st["past"]) + -(-L // BLOCK)
        ids, listed_ = ids[:, :used], listed_[:, :used]
    n = ids.shape[1]
    pages = torch.gather(table.to(torch.int64), 1, ids)
    K = _of_pages(st["kp"][pages.reshape(-1)], False).view(rows, n * BLOCK, D)
    V = _of_pages(st["vp"][pages.reshape(-1)], True).view(rows, n * BLOCK, D)
    kpos = (ids[..., None] * BLOCK + torch.arange(BLOCK, device=dev)).view(rows, n * BLOCK)
    there = listed_[..., None].expand(rows, n, BLOCK).reshape(rows, n * BLOCK)
    qr = q.float().view(B, L, H, G, D).permute(0, 2, 1, 3, 4).reshape(rows, L * G, D)
    s = torch.matmul(qr, K.transpose(1, 2)) * SCALE
    qpos = qpos0.repeat_interleave(H)[:, None] + torch.arange(L, device=dev).repeat_interleave(G)
    seen = there[:, None, :] & (kpos[:, None, :] <= qpos[:, :, None])
    s = s.masked_fill(~seen, float("-inf"))
    s = s - s.amax(-1, keepdim=True)
    p = torch.exp(s)
    o = torch.matmul(p, V) / p.sum(-1, keepdim=True)
    return o.view(B, H, L, G, D).permute(0, 2, 1, 3, 4).reshape(B, L, Hq, D).to(torch.bfloat16)


def _copy(st):
    dev = st["pools"][0].device
    src, dst = (torch.from_numpy(st[n]).to(dev, torch.int64) for n in ("src", "dst"))
    for pool in st["pools"]:
        pool[dst] = pool[src]
    return list(st["pools"])


def run(st):
    op = st["op"]
    if own:
        from compactattention_amd import ops

        if op == "norm_rope":
            return ops.norm_rope_qk(st["q"], st["k"], st["qw"], st["kw"], EPS, st["cos"], st["sin"])
        if op == "copy":
            ops.copy_pages(st["pools"], st["src"], st["dst"])
            return list(st["pools"])
        K, V = ops.KV4.paged(st["kp"], st["table"]), ops.KV4.paged(st["vp"], st["table"])
        if op == "append":
            B, L, H, _ = st["k"].shape
            ops.append_q4(st["k"], st["v"], K, V, st["starts"], st["cap"])
            return ops.gather_q4(K, V, B, H, st["starts"], L)
        H = st["table"].shape[0] // st["q"].shape[0]
        if op == "decode":
            return ops.attn_decode(st["q"], K, V, st["lens"], SCALE, st["cap"], H)
        return ops.attn_fwd(st["q"], K, V, st["blocks"], st["counts"], st["past"], SCALE, st["cap"], H)
    return {"norm_rope": _norm_rope, "append": _append, "copy": _copy, "decode": _attend, "chunk": _attend}[op](st)


# ----------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """(keys read over all KV rows, visible (row, key) pairs over all query heads) of an attention case."""
    L, hq, hkv = case["length"], case["hq"], case["hkv"]
    keys = pairs = 0
    if case["op"] == "decode":
        for n in _ints(case["lens"]):
            keys += n * hkv
            pairs += hq * sum(n - L + t + 1 for t in range(L))
    else:
        for p in _ints(case["past"]):
            kept = case["keep"] * p * BLOCK
            keys += (kept + L) * hkv
            pairs += hq * (L * kept + L * (L + 1) / 2)
    return keys, pairs


def work(case):
    op = case["op"]
    if op == "norm_rope":
        rows = case["batch"] * case["length"] * (case["hq"] + case["hkv"])
        return {"bytes": rows * 512 + case["length"] * 1024, "flops": rows * D * 9}
    if op == "append":
        rows = 2 * len(_ints(case["starts"])) * case["length"] * case["hkv"]
        return {"bytes": rows * (256 + 68 + 256), "flops": rows * D * 4}
    if op == "copy":
        page = PAGE if case["bits"] == 4 else BLOCK * D * 2
        return {"bytes": 2 * 2 * case["pages"] * page, "flops": 0}
    keys, pairs = _pairs(case)
    batch = len(_ints(case["lens"] if op == "decode" else case["past"]))
    return {"bytes": keys * 136 + 2 * batch * case["length"] * case["hq"] * 256, "flops": 4 * D * pairs}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _level64(code):
    """The value of E2M1 codes: sign, two exponent bits, one mantissa bit."""
    s = 1.0 - 2.0 * (code >> 3).double()
    e, m = ((code >> 1) & 3).double(), (code & 1).double()
    return s * torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)


def _token64(page, values):
    """[n, 4352] -> fp64 [n, 64, 128], each element looked up at its own byte."""
    t = torch.arange(BLOCK, device=page.device)[:, None]
    d = torch.arange(D, device=page.device)[None, :]
    g = d // 32
    if values:
        at, sat = 256 * (t // 4) + 16 * (d // 8) + 4 * (t % 4) + d % 8 // 2, 64 * g + 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4
    else:
        at, sat = 64 * t + d // 2, 64 * g + 4 * (t % 16) + t // 16
    byte = page[:, at].to(torch.int32)
    code = torch.where(d % 2 == 1, byte >> 4, byte & 15)
    return _level64(code) * torch.exp2(page[:, 4096 + sat].double() - 127)


def _quantised64(x):
    """The nearest level of every element at its group's scale (ties to the even code), fp64."""
    g = x.double().reshape(*x.shape[:-1], 4, 32)
    amax = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -122) / 7.0))
    e = torch.where(amax > 7.0 * torch.exp2(e), e + 1, e)  # log2's own rounding
    e = torch.where(amax <= 7.0 * torch.exp2(e - 1), e - 1, e).clamp(-125, 125)
    y = g / torch.exp2(e)
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.round(a / step) * step * torch.sign(y) * torch.exp2(e)).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        out = []
        c, s = st["cos"].double(), st["sin"].double()
        for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
            x = x.double()
            y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
            a, b = y[..., :D // 2], y[..., D // 2:]
            c0, c1, s0, s1 = (v[None, :, None] for v in (c[:, :D // 2], c[:, D // 2:], s[:, :D // 2], s[:, D // 2:]))
            out.append(torch.cat([a * c0 - b * s0, b * c1 + a * s1], -1))
        return tuple(out)
    if op == "append":
        return tuple(_quantised64(st[n].transpose(1, 2)) for n in ("k", "v"))
    if op == "copy":
        out = []
        for pool in st["pools"]:
            new = pool.clone()
            for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
                new[b].copy_(pool[a])
            out.append(new)
        return out
    q = st["q"]
    B, L, Hq, _ = q.shape
    H = case["hkv"]
    G = Hq // H
    out = torch.empty((B, L, Hq, D), dtype=torch.float64, device=q.device)
    for b in range(B):
        for h in range(H):
            r = b * H + h
            if op == "decode":
                first, ids = st["lens"][b] - L, torch.arange(-(-st["lens"][b] // BLOCK), device=q.device)
            else:
                first, ids = BLOCK * st["past"][b], st["blocks"][r, :int(st["counts"][r])].to(torch.int64)
            pages = st["table"][r, ids].to(torch.int64)
            k = _token64(st["kp"][pages], False).reshape(-1, D)
            v = _token64(st["vp"][pages], True).reshape(-1, D)
            kpos = (BLOCK * ids[:, None] + torch.arange(BLOCK, device=q.device)).reshape(-1)
            rows = q[b, :, h * G:(h + 1) * G].double()
            s = torch.matmul(rows.reshape(L * G, D), k.t()) / math.sqrt(D)
            hidden = kpos[None, :] > (first + torch.arange(L, device=q.device)).repeat_interleave(G)[:, None]
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[b, :, h * G:(h + 1) * G] = torch.matmul(p, v).view(L, G, D)
    return out
