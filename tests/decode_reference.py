"""Plain numpy forms, in 64 bits, of the one-token decode operators
(velo_cuda_kv_append, velo_cuda_decode_attention, velo_cuda_token_logprobs)."""
import numpy as np


def attention(q, k_pool, v_pool, table, lens, k_scale=None, v_scale=None, scale=None):
    """out [B][Hq][D], lse [B][Hq] and, for tolerances, the largest sum of
    |scale q_i k_i| of any score and the largest |v|."""
    B, Hq, D = q.shape
    Hkv = k_pool.shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out, lse = np.zeros((B, Hq, D)), np.full((B, Hq), -np.inf)
    reach, vmax = 0.0, 0.0
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        ids = table[b, :-(-n // 16)].astype(np.int64)

        def rows(pool, sc):
            x = pool[ids].astype(np.float64).transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n]
            if sc is None:
                return x
            return x * sc[ids].astype(np.float64).transpose(1, 0, 2).reshape(Hkv, -1)[:, :n, None]
        k, v = rows(k_pool, k_scale), rows(v_pool, v_scale)
        vmax = max(vmax, np.abs(v).max())
        for h in range(Hq):
            kh = k[h // (Hq // Hkv)]
            qh = q[b, h].astype(np.float64) * scale
            s = kh @ qh
            reach = max(reach, (np.abs(kh) @ np.abs(qh)).max())
            m = s.max()
            e = np.exp(s - m)
            lse[b, h] = m + np.log(e.sum())
            out[b, h] = (e / e.sum()) @ v[h // (Hq // Hkv)]
    return out, lse, reach, vmax


def rotate(x, pos, base):
    """NeoX half split of rows [T][H][D] at positions [T]."""
    D = x.shape[-1]
    a = pos.astype(np.float64)[:, None] * base ** (-2.0 * np.arange(D // 2) / D)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x0, x1 = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
    return np.concatenate((x0 * c - x1 * s, x0 * s + x1 * c), -1)


def logprobs(x, tokens, n, T):
    """logprob [M], entropy [M], top ids [M][n], top logprobs [M][n]."""
    with np.errstate(all="ignore"):
        M, V = x.shape
        s = x.astype(np.float64) / T
        m = s.max(-1, keepdims=True)
        d = s - np.where(np.isneginf(m), 0.0, m)
        e = np.exp(d)
        z = e.sum(-1, keepdims=True)
        bad = np.isnan(s).any(-1) | np.isposinf(s).any(-1)
        lp = np.where(np.isneginf(d), -np.inf, d - np.log(z))
        lp[bad] = np.nan
        ent = np.log(z[:, 0]) - np.where(e > 0, d * e, 0.0).sum(-1) / z[:, 0]
        ent = np.where(np.isneginf(m[:, 0]), 0.0, ent)
        ent[bad] = np.nan
        order = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
        top = np.empty((M, n), np.int64)
        for i in range(M):  # value descending, NaN below -inf, the lower index first
            top[i] = np.lexsort((np.arange(V), np.isnan(x[i]), -order[i]))[:n]
        return lp[np.arange(M), tokens], ent, top, np.take_along_axis(lp, top, 1)
