"""The 4-bit cache and what works on it, restated in 64 bits on the CPU: storage by the formulas of ``csrc/kv_cache.cuh``, written out
byte by byte, and attention row by row."""
import math

import numpy as np
import torch

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])


def stored(D):
    return 64 if D <= 64 else 128


def offsets(DS):
    """Byte offsets in a record of 16 tokens: key codes [16, DS/2], key scales [16, DS/16], and those of the values."""
    t = np.arange(16)[:, None]
    ch, b, S = np.arange(0, DS, 2)[None], np.arange(DS // 16)[None], DS // 64
    return (t * (DS // 2) + ch // 2,
            8 * DS + (4 * (t & 7) + b // S) * 2 * S + (t >> 3) * S + b % S,
            9 * DS + (t >> 3) * 4 * DS + ch // (DS // 8) * (DS // 2) + ((t >> 1) & 3) * (DS // 8) + (t & 1) * (DS // 16) + ch % (DS // 8) // 2,
            17 * DS + 16 * b + 4 * ((t >> 1) & 3) + 2 * (t >> 3) + (t & 1))


def nearest(x, grid):
    """Index of the nearest value of an ascending grid, the even one on a tie; x >= 0."""
    i = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo, hi = x - grid[i - 1], grid[i] - x
    return np.where((hi < lo) | ((hi == lo) & (i % 2 == 0)), i, i - 1)


def quantise(x):
    """float64 [..., 16 n] -> codes in 0 ... 15 [..., 16 n], scale bytes [..., n]; finite values."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    s = nearest(np.abs(b).max(-1) / 6, E4M3)
    sf = E4M3[s][..., None]
    y = np.divide(b, sf, out=np.zeros_like(b), where=sf > 0)
    code = nearest(np.abs(y), E2M1) + 8 * (np.signbit(b) & (sf > 0))
    return code.reshape(x.shape), s.astype(np.uint8)


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).double().numpy()


def write(data, page_size, slots, k, v, k_offset=None):
    """Writes bf16 [T, H, D] tokens to data uint8 [pages, H, bytes] (numpy, in place)."""
    T, H, D = k.shape
    DS = stored(D)
    k, v = k.double().numpy(), v.double().numpy()
    if k_offset is not None:
        k = bf16(k - k_offset.double().numpy())
    pad = ((0, 0), (0, 0), (0, DS - D))
    parts = []
    for x in (k, v):
        c, s = quantise(np.pad(x, pad))
        parts += [(c[..., 0::2] + 16 * c[..., 1::2]).astype(np.uint8), s]
    rec = data.reshape(data.shape[0], H, page_size // 16, 18 * DS)
    off = offsets(DS)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < data.shape[0] * page_size:
            place = s % page_size
            for p, o in zip(parts, off):
                rec[s // page_size, :, place // 16, o[place % 16]] = p[i].T


def values(data, D, page_size):
    """data uint8 [pages, H, bytes] -> keys (without offset) and values float64 [pages, H, page_size, D]."""
    DS = stored(D)
    P, H, _ = data.shape
    rec = data.reshape(P, H, page_size // 16, 18 * DS)
    table = np.concatenate((E2M1, -E2M1))
    scale = np.concatenate((E4M3, [np.nan]))
    scale = np.concatenate((scale, -scale))
    kc, ks, vc, vs = (rec[..., o] for o in offsets(DS))
    out = []
    for c, s in ((kc, ks), (vc, vs)):
        x = table[np.stack((c & 15, c >> 4), -1)].reshape(*c.shape[:-1], DS // 16, 16) * scale[s][..., None]
        out.append(x.reshape(P, H, page_size, DS)[..., :D])
    return out


def attend(q, data, D, page_size, table, kv_lens, q_lens, causal=True, scale=None, k_offset=None):
    """q bf16 [tokens, Hq, D] -> (out, lse, bound of |out|'s error, of |lse|'s) in float64.

    The bounds.  Codes times scales and queries are exact in the kernels.  A score is a sum of D products in fp32, each addition of which
    may lose a unit in the last place of the largest partial sum (2^-23): within e = D 2^-23 scale sum|q k| of the true one, so a
    weight is within 2 e.  Weights are rounded to fp16 with the largest at 2^6 or above: by 2^-11 of themselves or, below fp16's normal
    numbers, by half of its step there, 2^-25, which is 2^-31 of the largest.  The exponential is within
    2^-22 of its value and 2^-23 |s log2 e| (its argument is rounded), the output is rounded to bf16 (2^-8).  Sums of
    weights and of products with values are fp32 sums in a fixed order over up to n keys, split over 16 lanes' partial sums at least:
    (n / 16 + 64) 2^-23 relative to the sum of magnitudes."""
    kk, vv = values(data, D, page_size)
    Hq, H = q.shape[1], data.shape[1]
    g = Hq // H
    scale = D ** -0.5 if scale is None else scale
    qd = q.double().numpy()
    out, lse = np.zeros(qd.shape), np.full(qd.shape[:2], -np.inf)
    tol, ltol = np.zeros(qd.shape), np.zeros(qd.shape[:2])
    row = 0
    for b, (n, nq) in enumerate(zip(kv_lens, q_lens)):
        ids = [table[b][j // page_size] for j in range(n)]
        held = np.array([0 <= p < data.shape[0] for p in ids], bool)
        at = np.array([p if ok else 0 for p, ok in zip(ids, held)], int)
        place = np.arange(n) % page_size
        for t in range(nq):
            seen = held & ((np.arange(n) <= n - nq + t) if causal else True) if n else np.zeros(0, bool)
            if seen.any():
                k, v = kk[at[seen], :, place[seen]], vv[at[seen], :, place[seen]]     # [keys, H, D]
                for h in range(Hq):
                    x, kh, vh = qd[row, h], k[:, h // g], v[:, h // g]
                    s = kh @ x * scale
                    m = s.max()
                    p = np.exp(s - m)
                    l = p.sum()
                    p /= l
                    o = p @ vh
                    shift = 0.0 if k_offset is None else scale * float(x @ k_offset[h // g].double().numpy())
                    out[row, h], lse[row, h] = o, m + math.log(l) + shift
                    mag = scale * (np.abs(kh) @ np.abs(x))
                    e = D * 2.0 ** -23 * mag.max()
                    sums = (len(s) / 16 + 64) * 2.0 ** -23
                    arg = 2.0 ** -23 * (np.abs(s).max() + abs(m)) * 1.5
                    weight = 2 * e + 2.0 ** -22 + 2 * arg + 2 * sums
                    tol[row, h] = 2.0 ** -8 * np.abs(o) * 1.01 + (2.0 ** -11 + weight) * (p @ np.abs(vh)) + len(s) * 2.0 ** -31 / l * np.abs(vh).max() + 1e-30
                    off = 0.0 if k_offset is None else D * 2.0 ** -23 * scale * float(np.abs(x) @ np.abs(k_offset[h // g].double().numpy()))
                    ltol[row, h] = weight + 2.0 ** -21 * (abs(lse[row, h]) + abs(m) + abs(shift)) + off
            row += 1
    return out, lse, tol, ltol
