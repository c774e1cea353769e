"""Plain float64 forms of the serving step's operators (for the tests only): tree decode, cache append, sampling.

Written from the definitions, token by token on the CPU; they share no code with the kernels or with the
attention oracle.
"""
import math

import torch


def chain_of(parents, t):
    """The nodes from the root to t, or None for an absent node."""
    path = []
    while t >= 0:
        path.insert(0, t)
        p = int(parents[t])
        if not -1 <= p < t:
            return None
        t = p
    return path


def gather_rows(cache, table, b, n):
    """(Hkv, n, D): the first n rows of sequence b."""
    if table is None:
        return cache[b, :, :n]
    page = cache.shape[2]
    rows = [cache[int(table[b, r // page]), :, r % page] for r in range(n)]
    return torch.stack(rows, 1) if rows else cache.new_zeros(cache.shape[1], 0, cache.shape[3])


def decode_tree(q, k, v, k_cache, v_cache, lens, parents, table, lam, scale):
    """(o, lse, o_bound, lse_bound) in float64; parents (B, T) as nested lists or a tensor, or None for a chain.

    The bounds are how far fp32 arithmetic may take o and lse, to first order, before o is rounded to its
    type: with u = 2^-24, an exponent a_j = t_j - lam z_j is off by at most
      d_j = u * ((D + 12) * sum_d |q_d k_jd| * scale + (48 + n / 32) * lam * z_j + 8 * (|a_j| + |max a|) + 8)
    (a product of D terms in some order and its scale; sums of sigmoids over lanes, 16-key runs and 32-key
    tiles, each sigmoid within 6 u of its own; the roundings of the shifts and of the exponential), so the
    weight p_j is off by d_j of itself, o by sum_j p_j (d_j + e) (|v_j| + |o|) and lse by sum_j p_j d_j + 4 u (|lse| + 1), where e is
    what a weight may be rounded by for the product with V: half a step of the input type.
    """
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    e = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2
    u = 2.0 ** -24
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        kc, vc = gather_rows(k_cache, table, b, lens[b]), gather_rows(v_cache, table, b, lens[b])
        for t in range(T):
            path = list(range(t + 1)) if parents is None else chain_of(parents[b], t)
            if path is None:
                continue
            keys = torch.cat([kc, k[b][:, path]], 1).double().repeat_interleave(Hq // Hkv, 0)
            vals = torch.cat([vc, v[b][:, path]], 1).double().repeat_interleave(Hq // Hkv, 0)
            prod = q[b, :, t].double()[:, None] * keys
            x = prod.sum(2) * scale
            sig = torch.sigmoid(x)
            z = sig.flip(1).cumsum(1).flip(1)
            a = x - lam.double()[:, None] * z
            m = a.max(1, keepdim=True).values
            p = torch.softmax(a, 1)
            n = keys.shape[1]
            d = u * ((D + 12) * prod.abs().sum(2) * abs(scale) + (48 + n / 32) * lam.double()[:, None] * z
                     + 8 * (a.abs() + m.abs()) + 8)
            o[b, :, t] = (p[:, :, None] * vals).sum(1)
            lse[b, :, t] = torch.logsumexp(a, 1)
            ob[b, :, t] = (p[:, :, None] * (d + e + n * u)[:, :, None] * (vals.abs() + o[b, :, t][:, None].abs())).sum(1)
            lb[b, :, t] = (p * d).sum(1) + n * u + 4 * u * (lse[b, :, t].abs() + 1)
    return o, lse, ob, lb


def cache_append(k, v, k_cache, v_cache, lens, table, rows, counts):
    """The caches after the call (copies)."""
    out = [k_cache.clone(), v_cache.clone()]
    B, _, T, _ = k.shape
    page = k_cache.shape[2]
    capacity = page if table is None else page * table.shape[1]
    n = T if rows is None else rows.shape[1]
    for b in range(B):
        for i in range(n if counts is None else max(0, min(int(counts[b]), n))):
            src = i if rows is None else int(rows[b, i])
            at = int(lens[b]) + i
            if not (0 <= src < T and 0 <= at < capacity):
                continue
            unit = b if table is None else int(table[b, at // page])
            if not 0 <= unit < k_cache.shape[0]:
                continue
            for new, cache in zip((k, v), out):
                cache[unit, :, at % page if table is not None else at] = new[b, :, src]
    return out


def sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """Token of each row; the settings are one value per row (lists)."""
    out = []
    for b, row in enumerate(logits.double().tolist()):
        top = max(row) if not any(math.isnan(x) for x in row) else math.nan
        if math.isnan(top) or top == -math.inf:
            out.append(-1)
            continue
        order = sorted(range(len(row)), key=lambda i: (-row[i], i))
        t, u = temperature[b], float(uniforms[b])
        if not t > 0:
            out.append(order[0])
            continue
        if top_k[b] > 0:
            order = order[:top_k[b]]
        w = [1.0 if row[i] == top else 0.0 if row[i] == -math.inf or top == math.inf else math.exp((row[i] - top) / t)
             for i in order]
        total, before, kept = math.fsum(w), 0.0, []
        for x in w:
            if kept and ((top_p[b] < 1 and not before < top_p[b] * total) or (min_p[b] > 0 and not x >= min_p[b])):
                break
            kept.append(x)
            before += x
        want = min(max(u if u == u else 0.0, 0.0), 1.0) * math.fsum(kept)
        run, pick = 0.0, 0
        for j, x in enumerate(kept):
            run += x
            if x > 0:
                pick = j
            if run > want:
                break
        out.append(order[pick])
    return out
