"""Plain 64-bit restatements of the 4-bit cache's operators and of beam search,
written from the formulas in include/forgecu.h (numpy, no framework code)."""
import math

import numpy as np

PADS = (32, 64, 96, 128, 192, 256)


def row_bytes(dH):
    return next(p for p in PADS if p >= dH) // 2


def bf16(x):
    """fp32 rounded to bf16, ties to even, as fp32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
    return r.view(np.float32).reshape(np.shape(x))


def quantize(x):
    """(codes uint8, step, base) of rows x [..., dH] fp32."""
    x = np.asarray(x, np.float32)
    bad = ~(np.abs(x) < 2.0 ** 127).all(-1, keepdims=True)
    z = np.where(bad, np.float32(0), x)
    base = bf16(z.min(-1, keepdims=True)).astype(np.float64)
    step = bf16((np.maximum(z.max(-1, keepdims=True) - base, 0) / 15).astype(np.float32)).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        t = np.where(step > 0, (z.astype(np.float64) - base) / step, 0.0)
    code = np.clip(np.rint(t), 0, 15).astype(np.uint8)
    nan = np.where(bad, np.nan, 0.0)
    return code, step + nan, base + nan


def pack(code, rb):
    out = np.zeros((*code.shape[:-1], 2 * rb), np.uint8)
    out[..., :code.shape[-1]] = code
    return out[..., 0::2] | out[..., 1::2] << 4


def values(code, step, base):
    """What codes on a grid stand for, rounded once to fp32."""
    return (base + step * code).astype(np.float32)


def rope(x, pos, theta):
    """x [heads, dH] fp32 at position pos: interleaved pairs, fp32 table, rotation in double."""
    dH = x.shape[-1]
    ang = pos * (1.0 / np.power(theta, np.arange(0, dH, 2) / dH))
    c, s = np.cos(ang).astype(np.float32).astype(np.float64), np.sin(ang).astype(np.float32).astype(np.float64)
    u, v = x[:, 0::2].astype(np.float64), x[:, 1::2].astype(np.float64)
    out = np.empty_like(x)
    out[:, 0::2], out[:, 1::2] = (u * c - v * s).astype(np.float32), (u * s + v * c).astype(np.float32)
    return out


def attention(q, K, V, scale):
    """(out [dH], p [n]) of one head in 64 bits; zeros for no slots."""
    if len(K) == 0:
        return np.zeros(q.shape[-1]), np.zeros(0)
    s = scale * (K.astype(np.float64) @ q.astype(np.float64))
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ V.astype(np.float64), p


def evict(weight, pos, n, budget, recent):
    """(destination slots, source slots) of one head's moves."""
    if n <= budget:
        return np.zeros(0, int), np.zeros(0, int)
    w = np.where(np.isnan(weight[:n]), -np.inf, weight[:n].astype(np.float64))
    nan = np.isnan(weight[:n])
    safe = pos[:n].astype(np.int64) > int(pos[:n].max()) - recent
    order = sorted(range(n), key=lambda j: (not safe[j], nan[j] and not safe[j], 0 if safe[j] else -w[j], j))
    keep = np.zeros(n, bool)
    keep[order[:budget]] = True
    return np.flatnonzero(~keep[:budget]), budget + np.flatnonzero(keep[budget:])


def beam(logits, scores, done, W, eos):
    """One selection; logits [B, W, V]: (scores, tokens, parents, done) [B, W]."""
    B, _, V = logits.shape
    out = (np.zeros((B, W)), np.zeros((B, W), int), np.zeros((B, W), int), np.zeros((B, W), bool))
    for b in range(B):
        val = np.full((W, V), -np.inf)
        for w in range(W):
            x = logits[b, w].astype(np.float64)
            if done[b, w]:
                val[w, eos] = scores[b, w]
            elif np.isfinite(x.max()) and not np.isnan(x).any():
                lse = x.max() + math.log(np.exp(x - x.max()).sum())
                val[w] = float(scores[b, w]) + (x - lse)
        val[~np.isfinite(val)] = -np.inf
        flat = val.ravel()
        best = np.argsort(-flat, kind="stable")[:W]
        out[0][b], out[1][b], out[2][b] = flat[best], best % V, best // V
        out[3][b] = done[b][best // V] | (best % V == eos)
    return out
