"""Plain 64-bit statements of the 8-bit block-scaled KV cache and of packed
attention, written from the definitions in include/acefa.h (numpy, loops)."""
import numpy as np

BLOCK = 64


def rne(x):
    return np.rint(x)  # ties to even


def store(q, scale, new, pos, cu):
    """q (sets, H, n, D) int8 and scale (sets, H, nb) f32 after the store; new (H, rows, D) f32."""
    q, scale = q.copy(), scale.copy()
    n_max = q.shape[2]
    for s in range(q.shape[0]):
        a, b = int(cu[s]), int(cu[s + 1])
        p = int(pos[s])
        if a < 0 or b < a or b > new.shape[1] or (b > a and (p < 0 or p + b - a > n_max)):
            continue
        for blk in range(p // BLOCK, -(-(p + b - a) // BLOCK) if b > a else 0):
            lo, hi = max(blk * BLOCK, p), min(blk * BLOCK + BLOCK, p + b - a)
            for h in range(q.shape[1]):
                x = new[h, a + lo - p:a + hi - p]
                d = np.float32(np.abs(x).max()) / np.float32(127.0)
                if not np.isfinite(x).all():
                    d = np.float32(np.nan)
                old = scale[s, h, blk]
                keep = slice(blk * BLOCK, lo)
                if lo > blk * BLOCK:
                    if not (d <= old):  # grew (or NaN)
                        if d > old:
                            q[s, h, keep] = rne(q[s, h, keep].astype(np.float64) * np.float64(old) / np.float64(d))
                    else:
                        d = old
                if d > 0:
                    q[s, h, lo:hi] = np.clip(rne(x.astype(np.float64) / np.float64(d)), -127, 127)
                else:
                    q[s, h, lo:hi] = 0
                scale[s, h, blk] = d
    return q, scale


def values(q, scale, dtype=np.float64):
    n = q.shape[2]
    return q.astype(dtype) * np.repeat(scale, BLOCK, -1)[..., :n, None].astype(dtype)


def softmax_rows(s, visible):
    """Rows of weights; a row that sees nothing is zero."""
    s = np.where(visible, s, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    e = np.where(visible, np.exp(s - np.where(np.isinf(top), 0.0, top)), 0.0)
    total = e.sum(-1, keepdims=True)
    return e / np.where(total == 0, 1.0, total)


def attend(q, k, v, lens, scale):
    """q (sets, Hq, n_q, D), k, v (sets, H, n, D) f64: out (sets, n_q, Hq, D) and weights (sets, H, n)."""
    B, Hq, n_q, D = q.shape
    H, n = k.shape[1], k.shape[2]
    G = Hq // H
    out, w = np.zeros((B, n_q, Hq, D)), np.zeros((B, H, n))
    for b in range(B):
        ln = min(max(int(lens[b]), 0), n)
        i = np.arange(n_q)[:, None]
        vis = np.arange(ln)[None, :] < ln - (n_q - 1 - i)
        for hq in range(Hq):
            h = hq // G
            p = softmax_rows(q[b, hq] @ k[b, h, :ln].T * scale, vis)
            out[b, :, hq] = p @ v[b, h, :ln]
            w[b, h, :ln] += p.sum(0)
    return out, w


def evict(q, scale, weight, lens, keep, n_first, n_recent):
    """For one of K and V: (q, scale, kept, lens, weights) of the smaller cache."""
    B, H, n, D = q.shape
    nb = -(-keep // BLOCK)
    oq, os = np.zeros((B, H, keep, D), np.int8), np.zeros((B, H, nb), np.float32)
    kept, ow = np.full((B, H, keep), -1, np.int32), np.zeros((B, H, keep), np.float32)
    lo = np.zeros(B, np.int32)
    for b in range(B):
        ln = min(max(int(lens[b]), 0), n)
        m = min(ln, keep)
        lo[b] = m
        for h in range(H):
            if ln <= keep:
                at = np.arange(ln)
            else:
                mid = np.arange(n_first, ln - n_recent)
                w = weight[b, h, mid].astype(np.float64)
                w = np.where(np.isnan(w), -np.inf, w) + 0.0
                isnan = np.isnan(weight[b, h, mid])
                order = sorted(range(len(mid)), key=lambda t: (-w[t], isnan[t], t))
                at = np.sort(np.concatenate([np.arange(n_first), mid[order[:keep - n_first - n_recent]],
                                             np.arange(ln - n_recent, ln)])).astype(int)
            kept[b, h, :m] = at
            ow[b, h, :m] = weight[b, h, at]
            for blk in range(-(-m // BLOCK)):
                rows = at[blk * BLOCK:min(m, blk * BLOCK + BLOCK)]
                d = scale[b, h, rows // BLOCK]
                top = d.max()
                os[b, h, blk] = top
                x = q[b, h, rows].astype(np.float64) * d[:, None].astype(np.float64)
                oq[b, h, blk * BLOCK:blk * BLOCK + len(rows)] = rne(x / np.float64(top)) if top > 0 else q[b, h, rows]
    return oq, os, kept, lo, ow


def packed(q, k, v, cu_q, cu_k, mask, window, scale):
    """q (Hq, rows, D), k, v (H, rows_kv, D) f64 -> (rows, Hq, D); NaN where no sequence writes."""
    Hq, rows, D = q.shape
    G = Hq // k.shape[0]
    out = np.full((rows, Hq, D), np.nan)
    for s in range(len(cu_q) - 1):
        a, b, c, d = int(cu_q[s]), int(cu_q[s + 1]), int(cu_k[s]), int(cu_k[s + 1])
        n_q, n_k = b - a, d - c
        i, j = np.arange(n_q)[:, None], np.arange(n_k)[None, :]
        if mask == 1:
            vis = j <= i + n_k - n_q
        elif mask == 2:
            vis = np.abs(i - j) <= window
        else:
            vis = np.ones((n_q, n_k), bool)
        for h in range(Hq):
            p = softmax_rows(q[h, a:b] @ k[h // G, c:d].T * scale, vis)
            out[a:b, h] = p @ v[h // G, c:d]
    return out
