"""float64 CPU restatement of the paged cache's operators (dark_amd/kv_cache.py), written from their definitions, for
the tests only.  The attention also returns the bound its caller derives tolerances from."""
import math

import torch


def norm_rope(x, w, cos, sin, pos, eps):
    """x [T, H, D] -> (y, a): y = rope(w * x / rms(x)) and a = |first term| + |second term| of the rotation, in float64."""
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is None:
        return x, x.abs()
    p = pos.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    a = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
    return y, a


def append(cache, rows, slots):
    """cache [pages, page, H, D]; later tokens are not needed to win: slots differ."""
    out = cache.clone()
    pages, page = cache.shape[:2]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            out[s // page, s % page] = rows[t]
    return out


def attention(q, k_cache, v_cache, table, cu_q, kv_len, q_index=None, key_mask=None, causal=False, scale=None):
    """(out, lse, a, z): out [T, H, D] and lse [T, H] in float64 (zeros / -inf for a token with no key; tokens of no
    sequence stay NaN); a = sum_j p_j |v_j| and z = scale * max_j sum_i |q_i k_ji|, what rounding errors are measured in."""
    T, H, D = q.shape
    pages, page, Hk, _ = k_cache.shape
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, H), math.nan, dtype=torch.float64)
    a = torch.zeros(T, H, D, dtype=torch.float64)
    z = torch.zeros(T, H, dtype=torch.float64)
    for b in range(len(kv_len)):
        t0, t1 = int(cu_q[b]), int(cu_q[b + 1])
        n = max(0, min(int(kv_len[b]), table.shape[1] * page))
        keys = []
        for j in range(n):
            p = int(table[b, j // page])
            if 0 <= p < pages and (key_mask is None or bool(key_mask[b, j])):
                keys.append((j, p, j % page))
        js = torch.tensor([x[0] for x in keys], dtype=torch.long)
        K = k_cache[[x[1] for x in keys], [x[2] for x in keys]].double()     # [m, Hk, D]
        V = v_cache[[x[1] for x in keys], [x[2] for x in keys]].double()
        for t in range(t0, t1):
            at = int(q_index[t]) if q_index is not None else int(kv_len[b]) - (t1 - t)
            sel = (js <= at) if causal else torch.ones(len(keys), dtype=torch.bool)
            m = int(sel.sum())
            if m == 0:
                out[t], lse[t] = 0.0, -math.inf
                continue
            Kt, Vt = K[sel].repeat_interleave(G, 1), V[sel].repeat_interleave(G, 1)
            qt = q[t].double()
            s = (Kt * qt).sum(-1) * scale                                     # [m, H]
            z[t] = ((Kt.abs() * qt.abs()).sum(-1) * abs(scale)).amax(0)
            lse[t] = s.logsumexp(0)
            p = (s - lse[t]).exp()
            out[t] = (p[..., None] * Vt).sum(0)
            a[t] = (p[..., None] * Vt.abs()).sum(0)
    return out, lse, a, z
