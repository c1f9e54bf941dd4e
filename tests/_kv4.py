"""The 4-bit key/value cache restated for the tests, on the CPU: the format in numpy fp32 (its definition's
arithmetic), its bytes, and attention over it in 64 bits."""
from __future__ import annotations

import numpy as np
import torch


def page_bytes(P, D, G):
    return P * (D + 8 * D // G)


def quantise(x, G):
    """x [..., D] fp32 -> codes uint8 [..., D], scales and zeros fp16 [..., D/G]."""
    w = np.clip(x.astype(np.float32), np.float32(-65504), np.float32(65504)).reshape(*x.shape[:-1], -1, G)
    lo, hi = w.min(-1), w.max(-1)
    with np.errstate(invalid="ignore"):
        step = np.maximum(np.maximum((hi - lo) / np.float32(15), np.maximum(np.abs(lo), np.abs(hi)) / np.float32(96)), np.float32(2.0**-14))
        s = step.astype(np.float16)
        z = (np.rint(-lo / s.astype(np.float32) * np.float32(8)) / np.float32(8)).astype(np.float16)
        q = np.clip(np.rint(w / s.astype(np.float32)[..., None] + z.astype(np.float32)[..., None]), 0, 15)
    bad = np.isnan(w).any(-1)
    q[bad] = 0
    s[bad] = z[bad] = np.nan
    return q.astype(np.uint8).reshape(x.shape), s, z


def _place(t):
    return t // 16, t % 16 // 4 * 4 + (0, 2, 1, 3)[t % 4]


def write(cache, k, v, slots, G, P):
    """numpy uint8 cache [pages, H, bytes]; k, v fp32 [T, H, D]."""
    D = k.shape[-1]
    half, ng = D // 2, D // G
    pages = cache.shape[0]
    (qk, sk, zk), (qv, sv, zv) = quantise(k, G), quantise(v, G)
    pack = lambda q: q[..., :half] | (q[..., half:] << 4)  # noqa: E731
    bk, bv = pack(qk), pack(qv)
    for i, slot in enumerate(slots):
        if not 0 <= slot < pages * P:
            continue
        page, t = divmod(int(slot), P)
        tile, place = _place(t)
        for h in range(cache.shape[1]):
            c = cache[page, h]
            c[t * half:(t + 1) * half] = bk[i, h]
            c[P * half + tile * half * 16 + place:P * half + (tile + 1) * half * 16:16] = bv[i, h]
            side = c[P * D:].view(np.uint16).reshape(4, ng, P)
            for n, a in enumerate((sk, zk, sv, zv)):
                side[n, :, t] = np.where(np.isnan(a[i, h]), np.uint16(0x7E00), a[i, h].view(np.uint16))


def read(cache, slots, D, G, P):
    """(k, v) float64 [T, H, D]: the values that the bytes stand for, zeros for slots outside the cache."""
    half, ng, H = D // 2, D // G, cache.shape[1]
    out = np.zeros((2, len(slots), H, D))
    for i, slot in enumerate(slots):
        if not 0 <= slot < cache.shape[0] * P:
            continue
        page, t = divmod(int(slot), P)
        tile, place = _place(t)
        for h in range(H):
            c = cache[page, h]
            side = c[P * D:].view(np.float16).astype(np.float64).reshape(4, ng, P)[:, :, t]
            for n, b in enumerate((c[t * half:(t + 1) * half], c[P * half + tile * half * 16 + place:P * half + (tile + 1) * half * 16:16])):
                q = np.concatenate([b & 15, b >> 4]).astype(np.float64).reshape(ng, G)
                out[n, i, h] = ((q - side[2 * n + 1][:, None]) * side[2 * n][:, None]).reshape(D)
    return out[0], out[1]


def attention(q, cache, table, lens, G, P, q_start=None, scale=None, causal=True, window=0):
    """(out, lse, spread) in 64 bits: spread is the sum of p |v| over the sum of p, which errors scale with."""
    q = q.double().numpy()
    T, Hq, D = q.shape
    H = cache.shape[1]
    scale = D**-0.5 if scale is None else scale
    start = range(len(lens) + 1) if q_start is None else [int(x) for x in q_start]
    out, spread, lse = np.zeros(q.shape), np.zeros(q.shape), np.full((T, Hq), -np.inf)
    for b, n in enumerate(int(x) for x in lens):
        n = min(max(n, 0), table.shape[1] * P)
        m = start[b + 1] - start[b]
        page = np.array([int(table[b, t // P]) for t in range(n)], dtype=np.int64)
        there = (page >= 0) & (page < cache.shape[0])
        k, v = read(cache, np.where(there, page * P + np.arange(n) % P, -1), D, G, P)
        for i in range(m):
            pos = n - m + i
            t = np.arange(n)
            see = there & ((t <= pos) if causal else (t >= 0)) & ((t > pos - window) if window else (t >= 0))
            if not see.any():
                continue
            for h in range(Hq):
                kh, vh = k[see][:, h // (Hq // H)], v[see][:, h // (Hq // H)]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kh @ q[start[b] + i, h] * scale
                    p = np.exp(x - x.max())
                    out[start[b] + i, h], spread[start[b] + i, h] = p @ vh / p.sum(), p @ np.abs(vh) / p.sum()
                    lse[start[b] + i, h] = np.log(p.sum()) + x.max()
    return out, lse, spread


def bits(t):
    """A tensor's 16-bit patterns on the host."""
    return t.detach().cpu().contiguous().view(torch.int16).numpy()
