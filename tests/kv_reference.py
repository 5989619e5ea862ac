"""The paged key-value cache's operators in 64 bits, sequence by sequence, and the distance a correct kernel keeps from them."""
import numpy as np
import torch

U = 2.0 ** -24      # half a step of fp32, relative


def rows_of(pages, table, b, h, n):
    """The first n rows of sequence b, kv head h, in 64 bits."""
    page = pages.shape[2]
    ids = table[b, :-(-n // page)].long()
    return pages[ids, h].reshape(-1, pages.shape[3])[:n].double().cpu().numpy()


def attend(q, k_pages, v_pages, table, lengths, scale):
    """out [B, hq, d], lse [B, hq], weights (list of [hkv, L] summed over a kv head's query heads), and the tolerances of
    the three.

    A score is a sum of d products, exact in 32 bits for 16-bit inputs: rounding errors of a sum of n terms are independent,
    so 8 sqrt(n) U times the sum of magnitudes is an eight-sigma bound. Scaling, the subtraction of the maximum and the
    conversion to base 2 add a few U of the score's size, the exponential a step. A weight is off by that much,
    relatively, and by the normalising sum's 8 sqrt(L) U; where weights are split into two 16-bit halves for the second
    product, by 2^-16 more. The output is then rounded to its type: half a step."""
    B, hq, d = q.shape
    hkv = k_pages.shape[1]
    g = hq // hkv
    half = 2.0 ** -16 if q.dtype != torch.float32 else 0.0
    eps = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * eps
    out, out_tol = np.zeros((B, hq, d)), np.zeros((B, hq, d))
    lse, lse_tol = np.full((B, hq), -np.inf), np.zeros((B, hq))
    weights, w_tol = [], []
    qd = q.double().cpu().numpy()
    for b, L in enumerate(int(x) for x in lengths):
        w, wt = np.zeros((hkv, L)), np.zeros((hkv, L))
        for i in range(hq if L else 0):
            h = i // g
            k, v = rows_of(k_pages, table, b, h, L), rows_of(v_pages, table, b, h, L)
            s = (k @ qd[b, i]) * scale
            m = s.max()
            e = np.exp(s - m)
            total = e.sum()
            p = e / total
            ds = abs(scale) * (np.abs(k) @ np.abs(qd[b, i])).max() * 8 * np.sqrt(d) * U + 8 * U * np.abs(s).max() + 4 * U
            dp = ds + 8 * np.sqrt(L) * U + 4 * U
            out[b, i] = p @ v
            out_tol[b, i] = np.abs(v).max() * (2 * dp + half) + np.abs(out[b, i]) * eps + tiny
            lse[b, i] = m + np.log(total)
            lse_tol[b, i] = 2 * dp + 4 * U * abs(lse[b, i])
            w[h] += p
            wt[h] += p * 2 * dp + 2.0 ** -120       # (below 2^-126 a weight is flushed to 0)
        weights.append(w)
        w_tol.append(wt)
    return out, out_tol, lse, lse_tol, weights, w_tol


def survivors(mass, pos, n, recent):
    """Slots of one head that are kept, ascending: the newest `recent` positions (by slot, should positions repeat and more
    than n be among them), then the greatest masses (NaN greatest, equal ones by slot)."""
    L = len(mass)
    if n == L:
        return np.arange(L)
    new = pos.astype(np.int64) > int(pos.max()) - recent
    m = np.where(np.isnan(mass) | new, np.inf, mass.astype(np.float64))
    return np.sort(np.lexsort((np.arange(L), -m, ~(np.isnan(mass) | new), ~new))[:n])


def evict(k, v, mass, pos, lengths, budget, recent):
    """k, v: [B, hkv, slots, d] (numpy, any type), mass, pos [B, hkv, slots]. Returns copies after the eviction, lengths."""
    k, v = k.copy(), v.copy()
    new_mass, new_pos, new_len = np.zeros_like(mass), np.full_like(pos, -1), []
    for b, L in enumerate(int(x) for x in lengths):
        n = min(L, budget)
        new_len.append(n)
        for h in range(mass.shape[1]):
            keep = survivors(mass[b, h, :L], pos[b, h, :L], n, recent)
            src = np.arange(n)
            gaps = np.setdiff1d(src, keep)
            src[gaps] = keep[keep >= n]
            k[b, h, :n], v[b, h, :n] = k[b, h, src], v[b, h, src]
            new_mass[b, h, :n], new_pos[b, h, :n] = mass[b, h, src], pos[b, h, src]
    return k, v, new_mass, new_pos, np.array(new_len, np.int32)
