"""A 4-bit KV cache, page copies and the q/k norm with rotation in 64 bits, written from their definitions."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 4352
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def bf16(x) -> np.ndarray:
    """Nearest bf16 values as fp64."""
    return torch.as_tensor(np.asarray(x, np.float32)).to(torch.bfloat16).to(torch.float64).numpy()


def quantise(x: np.ndarray):
    """fp64 [..., 128] of bf16 values -> (codes uint8 [..., 128], scale bytes uint8 [..., 4]): per group of 32 the
    smallest power of two 2^(byte - 127), byte in [2, 252], under which the largest magnitude is at most 7; the
    nearest level, of two the one of even code; byte 255 and codes 0 for a group that is not finite."""
    g = x.reshape(*x.shape[:-1], 4, 32)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(np.isfinite(g), g, 0.0)
    amax = np.abs(g).max(-1)
    m, e = np.frexp(amax)  # amax = m 2^e, m in [1/2, 1): at most 7 * 2^(e - 3) exactly where m <= 7/8
    byte = np.where(amax == 0.0, 2, np.clip(np.where(m <= 0.875, e - 3, e - 2) + 127, 2, 252))
    y = g / 2.0 ** (byte[..., None].astype(np.float64) - 127)
    d = np.abs(np.abs(y)[..., None] - LEVELS)
    # the nearest level; of two equally near the even code (codes order as levels)
    near = d.min(-1, keepdims=True)
    tie = (d == near) & (np.arange(8) % 2 == 0)
    code = np.where(tie.any(-1), tie.argmax(-1), (d == near).argmax(-1)).astype(np.uint8)
    code = np.where(np.abs(y) >= 6.0, np.uint8(7), code)
    code = code | (np.signbit(y).astype(np.uint8) << 3)
    code = np.where(bad[..., None], np.uint8(0), code).astype(np.uint8)
    byte = np.where(bad, 255, byte).astype(np.uint8)
    return code.reshape(x.shape), byte


def values(code: np.ndarray, byte: np.ndarray) -> np.ndarray:
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return (v.reshape(*code.shape[:-1], 4, 32) * s[..., None]).reshape(code.shape)


def code_at(t: int, d: int, of_v: bool) -> int:
    return 256 * (t // 4) + 16 * (d // 8) + 4 * (t % 4) + d % 8 // 2 if of_v else 64 * t + d // 2


def scale_at(t: int, g: int, of_v: bool) -> int:
    return 4096 + 64 * g + (16 * (t % 16 // 4) + 4 * (t // 16) + t % 4 if of_v else 4 * (t % 16) + t // 16)


def write_token(page: np.ndarray, t: int, code: np.ndarray, byte: np.ndarray, of_v: bool) -> None:
    """Token t's codes [128] and scale bytes [4] into a page (uint8 [4352])."""
    for d in range(0, 128, 2):
        page[code_at(t, d, of_v)] = code[d] | (code[d + 1] << 4)
    for g in range(4):
        page[scale_at(t, g, of_v)] = byte[g]


_T, _D = np.arange(64)[:, None], np.arange(128)[None, :]
_CODE = {v: np.vectorize(lambda t, d, v=v: code_at(t, d, v))(_T, _D) for v in (False, True)}
_SCALE = {v: np.vectorize(lambda t, g, v=v: scale_at(t, g, v))(_T, np.arange(4)[None, :]) for v in (False, True)}


def read_pages(pages: torch.Tensor, of_v: bool) -> torch.Tensor:
    """uint8 [n, 4352] (any device) -> fp64 values [n, 64, 128] on it."""
    dev = pages.device
    at = torch.as_tensor(_CODE[of_v], device=dev)
    sat = torch.as_tensor(_SCALE[of_v], device=dev)
    w = pages[:, at].to(torch.int64)
    odd = torch.arange(128, device=dev) % 2 == 1
    code = torch.where(odd, w >> 4, w & 15)
    level = torch.tensor(np.concatenate([LEVELS, -LEVELS]), device=dev, dtype=torch.float64)
    byte = pages[:, sat].to(torch.float64)
    scale = torch.where(byte == 255, torch.full_like(byte, math.nan), torch.exp2(byte - 127))
    return level[code] * scale.repeat_interleave(32, dim=-1)


def make_pages(x: torch.Tensor, of_v: bool) -> torch.Tensor:
    """bf16 tokens [n, 64, 128] on the CPU -> pages uint8 [n, 4352]."""
    code, byte = quantise(x.double().numpy())
    out = np.zeros((x.shape[0], PAGE), np.uint8)
    out[:, _CODE[of_v][:, 0::2]] = code[..., 0::2] | (code[..., 1::2] << 4)
    out[:, _SCALE[of_v]] = byte
    return torch.from_numpy(out)


def attention(q, k, v, kpos, qpos, scale):
    """One KV row in 64 bits: q [R, 128], k and v [N, 128], positions kpos [N], qpos [R]: a query sees the keys at or
    before its position.  Hidden keys are left out altogether.  Returns (out [R, 128], lse [R], A [R, 128] = the
    weighted mean of |v|, S [R] = the largest sum of |q k| * scale over the keys a row sees)."""
    R = q.shape[0]
    out = torch.zeros((R, 128), dtype=torch.float64, device=q.device)
    lse = torch.full((R,), -math.inf, dtype=torch.float64, device=q.device)
    A, S = torch.zeros_like(out), torch.zeros_like(lse)
    for p in torch.unique(qpos).tolist():
        rows = (qpos == p).nonzero()[:, 0]
        seen = kpos <= p
        kk, vv = k[seen], v[seen]
        if kk.shape[0] == 0:
            continue
        s = (q[rows] @ kk.t()) * scale
        w = torch.softmax(s, -1)
        out[rows] = w @ vv
        lse[rows] = torch.logsumexp(s, -1)
        A[rows] = w @ vv.abs()
        S[rows] = (q[rows].abs() @ kk.abs().t()).amax(-1) * scale
    return out, lse, A, S


def tolerance(out, A, S, splits=1):
    """How far a bf16 output may be off.  Scores: 128 products and sums in fp32 in any order, the scale and the
    exponent's argument, 132 roundings of at most 2^-24 of S, in both the weight and the largest score; exp2 and the
    sums of an online softmax (a rounding per block and split) 2^-15 together.  The weights are rounded to bf16 (2^-8
    of each), the sum is that of the rounded weights, so an error e of every weight moves the output by at most
    e (A + |out|); the output is rounded to bf16 (2^-8, and half the smallest normal step)."""
    e = 2 * 132 * 2.0 ** -24 * S[:, None] * 1.4427 + 2.0 ** -15 + 2.0 ** -8
    return 1.02 * e * (A + out.abs()) + 2.0 ** -8 * out.abs() + 2.0 ** -126


def lse_tolerance(S):
    """The lse: the scores' error, and the sum of weights rounded by 2^-8 each (log(1 + x) <= 1.004 x here)."""
    return 2 * 132 * 2.0 ** -24 * S * 1.4427 + 1.01 * 2.0 ** -8 + 2.0 ** -15
