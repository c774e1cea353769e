"""Plain float64 forms of the 8-bit cache's and beam search's operators (for the tests only).

Written from the definitions, row by row on the CPU; they share no code with the kernels.
"""
import math

import torch

from .serving import chain_of

BLOCK = 16
LEAST, MOST = 2.0 ** -40, 2.0 ** 40
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def code(x, fmt):
    """The nearest codes of x (float64), as float64: ties to even."""
    if fmt == torch.int8:
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def append(k, v, caches, scales, lens, table, rows, counts):
    """(caches, scales) after the call: copies, the codes in the caches' dtype."""
    fmt = caches[0].dtype
    codes, scales = [c.to(torch.float64) for c in caches], [s.clone() for s in scales]
    B, Hkv, T, _ = k.shape
    units, _, page, _ = caches[0].shape
    capacity = page if table is None else page * table.shape[1]
    n = T if rows is None else rows.shape[1]
    for b in range(B):
        m = n if counts is None else max(0, min(int(counts[b]), n))
        first = int(lens[b])
        new = {}  # cache row -> new row
        for i in range(m):
            src, at = i if rows is None else int(rows[b, i]), first + i
            if 0 <= src < T and 0 <= at < capacity:
                new[at] = src
        for block in sorted({at // BLOCK for at in new}):
            at0 = block * BLOCK
            unit, base = (b, at0) if table is None else (int(table[b, at0 // page]), at0 % page)
            if not 0 <= unit < units:
                continue
            mine = [at for at in new if at // BLOCK == block]
            held = max(0, min(min(first, capacity) - at0, BLOCK))
            for c, s, x in zip(codes, scales, (k, v)):
                for h in range(Hkv):
                    y = torch.stack([x[b, h, new[at]].double() for at in mine])
                    top = float(y.abs().max()) if torch.isfinite(y).all() else math.inf
                    was = float(s[unit, h, base // BLOCK]) if held else LEAST
                    now = was
                    if not LEAST <= was <= MOST or top > LARGEST[fmt] * MOST:
                        now = math.nan
                    else:
                        while top > LARGEST[fmt] * now:
                            now *= 2
                        if now > MOST:
                            now = math.nan
                    s[unit, h, base // BLOCK] = now
                    if now == now and now != was:
                        c[unit, h, base:base + held] = code(c[unit, h, base:base + held] * (was / now), fmt)
                    for at, z in zip(mine, y):
                        c[unit, h, base + at - at0] = code(z / now, fmt) if now == now else 0.0
    return [c.to(fmt) for c in codes], scales


def values(cache, scale):
    """A cache's values in float64; NaN in blocks whose scale is none."""
    s = scale.double()
    s = torch.where((s >= LEAST) & (s <= MOST), s, math.nan)
    return cache.to(torch.float64) * s.repeat_interleave(BLOCK, 2)[:, :, :cache.shape[2], None]


def rows_of(vals, table, b, first, n):
    """(Hkv, n, D): cache rows first .. first + n of sequence b; NaN on a page outside the pool."""
    if table is None:
        return vals[b, :, first:first + n]
    page = vals.shape[2]
    out = [vals.new_zeros(vals.shape[1], 0, vals.shape[3])]
    for r in range(first, first + n):
        unit = int(table[b, r // page])
        out.append(vals[unit, :, r % page, None] if 0 <= unit < vals.shape[0]
                   else vals.new_full((vals.shape[1], 1, vals.shape[3]), math.nan))
    return torch.cat(out, 1)


def read(caches, scales, lens, table, first, rows):
    """k and v (B, Hkv, rows, D) in float64."""
    out = []
    capacity = caches[0].shape[2] * (1 if table is None else table.shape[1])
    for c, s in zip(caches, scales):
        vals = values(c, s)
        x = torch.zeros(len(lens), c.shape[1], rows, c.shape[3], dtype=torch.float64)
        for b in range(len(lens)):
            for i in range(rows):
                r = (0 if first is None else int(first[b])) + i
                if 0 <= r < min(int(lens[b]), capacity):
                    x[b, :, i] = rows_of(vals, table, b, r, 1)[:, 0]
        out.append(x)
    return out


def decode_tree(q, k, v, caches, scales, lens, parents, table, lam, scale):
    """(o, lse, o_bound, lse_bound) in float64, as oracle.serving.decode_tree.

    The bound has that one's terms, and of the scales of V: each exponent a_j + log2 vs is larger by up to |log2 vs|, which its
    roundings go by, and 1 / vs is one more.  The largest folded weight 2^(a_j + log2 vs - m) is at least 1, and small ones have an
    absolute error, too: half of fp16's smallest step, 2^-25, where they are rounded to fp16; else they become 0 below fp32's
    (and bf16's) smallest normal number, 2^-126.
    """
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    e = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2
    u = 2.0 ** -24
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(o), torch.zeros_like(lse)
    kv, vv = values(caches[0], scales[0]), values(caches[1], scales[1])
    vs_all = scales[1].double()
    for b in range(B):
        n0 = int(lens[b])
        kc, vc = rows_of(kv, table, b, 0, n0), rows_of(vv, table, b, 0, n0)
        units = [b] if table is None else [x for x in table[b, :-(-n0 // kv.shape[2])].tolist() if 0 <= x < kv.shape[0]]
        vs = torch.cat([vs_all[x] for x in units], 1)[:, :-(-n0 // BLOCK)] if n0 else torch.ones(Hkv, 1, dtype=torch.float64)
        shift = vs.log2().abs().amax(1).repeat_interleave(Hq // Hkv)[:, None]
        vs_most = vs.amax(1).clamp(min=1.0).repeat_interleave(Hq // Hkv)[:, None]
        vs_least = vs.amin(1).clamp(max=1.0).repeat_interleave(Hq // Hkv)[:, None]
        for t in range(T):
            path = list(range(t + 1)) if parents is None else chain_of(parents[b], t)
            if path is None:
                continue
            keys = torch.cat([kc, k[b][:, path].double()], 1).repeat_interleave(Hq // Hkv, 0)
            vals = torch.cat([vc, v[b][:, path].double()], 1).repeat_interleave(Hq // Hkv, 0)
            prod = q[b, :, t].double()[:, None] * keys
            x = prod.sum(2) * scale
            sig = torch.sigmoid(x)
            z = sig.flip(1).cumsum(1).flip(1)
            a = x - lam.double()[:, None] * z
            m = a.max(1, keepdim=True).values
            p = torch.softmax(a, 1)
            n = keys.shape[1]
            d = u * ((D + 12) * prod.abs().sum(2) * abs(scale) + (48 + n / 32) * lam.double()[:, None] * z
                     + 8 * (a.abs() + m.abs() + shift) + 10)
            o[b, :, t] = (p[:, :, None] * vals).sum(1)
            lse[b, :, t] = torch.logsumexp(a, 1)
            ob[b, :, t] = (p[:, :, None] * (d + e + n * u)[:, :, None] * (vals.abs() + o[b, :, t][:, None].abs())).sum(1)
            # A weight's error times its code |v_j| / vs_j, over a sum that is at least 1 / vs of the largest weight's key.
            smallest = 2.0 ** (-25 if q.dtype == torch.float16 else -126)
            ob[b, :, t] += smallest * (vs_most / vs_least) * vals.abs().sum(1)
            lb[b, :, t] = (p * d).sum(1) + n * u + 4 * u * (lse[b, :, t].abs() + shift[:, 0] + 1)
    return o, lse, ob, lb


def beam_select(logits, scores, num_beams, finished=None, end_token=0):
    """(scores, parents, tokens) as nested lists, scores in float64."""
    out = ([], [], [])
    for b in range(logits.shape[0]):
        found = []
        for w in range(logits.shape[1]):
            s = float(scores[b, w])
            if not math.isfinite(s):
                continue
            if finished is not None and bool(finished[b, w]):
                found.append((-s, w, 0.0, end_token))
                continue
            x = logits[b, w].double()
            top = float(x.max()) if not bool(x.isnan().any()) else math.nan
            if math.isnan(top) or top == -math.inf:
                continue
            if top == math.inf:
                n = int((x == top).sum())
                found += [(math.log(n) - s, w, 0.0, int(t)) for t in (x == top).nonzero()[:num_beams, 0]]
                continue
            below = math.log(math.fsum(torch.exp(x - top).tolist()))
            best = sorted((-float(x[t]), int(t)) for t in torch.topk(x, min(len(x), num_beams)).indices)
            least = -best[-1][0]  # all that tie with the last one
            best = sorted({(-float(x[t]), int(t)) for t in (x >= least).nonzero()[:, 0]})[:num_beams]
            found += [(-(s + ((-y - top) - below)), w, y, t) for y, t in best if y < math.inf]
        found = sorted(found)[:num_beams]
        found += [(math.inf, 0, 0.0, -1)] * (num_beams - len(found))
        out[0].append([-f[0] for f in found])
        out[1].append([f[1] for f in found])
        out[2].append([f[3] for f in found])
    return out


def reorder(caches, table, pages, lens, parents, page):
    """(caches, table, lens) after the call: copies."""
    B, W = parents.shape
    J = table.shape[1]
    out_table, out_lens = table.clone(), lens.clone()
    moves = []
    for g in range(B):
        par = [min(max(int(p), 0), W - 1) for p in parents[g]]
        n = [int(lens[g * W + p]) for p in par]
        for i in range(W):
            out_lens[g * W + i] = n[i]
        for j in range(J):
            held = [int(table[g * W + p, j]) for p in par]
            fill = [max(0, min(page, x - j * page)) for x in n]
            kept = {held[i] for i in range(W) if fill[i] == page}
            stay = [fill[i] == page for i in range(W)]
            for i in range(W):
                if 0 < fill[i] < page and held[i] not in kept:
                    kept.add(held[i])
                    stay[i] = True
            free = [int(pages[g * W + i, j]) for i in range(W) if int(pages[g * W + i, j]) not in kept]
            for i in range(W):
                out_table[g * W + i, j] = held[i] if stay[i] else free.pop(0)
                if not stay[i] and fill[i]:
                    moves.append((held[i], int(out_table[g * W + i, j]), fill[i]))
    out = [c.clone() for c in caches]
    for old, new in zip(caches, out):
        per = page // old.shape[2]
        for a, b, rows in moves:
            if 0 <= a < old.shape[0] and 0 <= b < old.shape[0]:
                new[b, :, :-(-rows // per)] = old[a, :, :-(-rows // per)]
    return out, out_table, out_lens


def check_search(logits_after, b, prompt, tokens, scores, steps, tol, end_token=None):
    """Asserts that a beam search did what it says.  ``steps``: its (scores, parents, tokens), batch entry ``b`` of which is checked.

    Every step's beams are the best of what ``logits_after(tokens)`` gives behind the step before's, up to ``tol`` on either side of
    a log probability (a logit's own and the sum's), and the result (tokens (W, n), scores (W,)) is the way back from the last.
    """
    W = tokens.shape[0]
    beams = [(0.0, [], False)]
    for s, p, t in steps:
        found = {}
        for w, (score, seq, done) in enumerate(beams):
            if done:
                found[w, end_token] = score
            elif math.isfinite(score):
                logp = torch.log_softmax(logits_after(prompt + seq), 0)
                found.update({(w, i): score + logp[i].item() for i in range(len(logp))})
        keys = [(p[b, i].item(), t[b, i].item()) for i in range(W) if s[b, i] > -math.inf]
        assert len(keys) == min(W, len(found)) == len(set(keys))
        got = s[b, :len(keys)].tolist()
        assert got == sorted(got, reverse=True)
        for key, score in zip(keys, got):
            assert abs(found[key] - score) <= 2 * tol + 2.0 ** -24 * abs(score)
        left = [f for key, f in found.items() if key not in keys]
        assert max(left, default=-math.inf) <= got[-1] + 2 * tol + 2.0 ** -24 * abs(got[-1])
        beams = [(score, beams[w][1] + [i], beams[w][2] or i == end_token) for (w, i), score in zip(keys, got)]
        beams += [(-math.inf, [], False)] * (W - len(beams))
    for i, (score, seq, _) in enumerate(beams):
        assert scores[i].item() == score
        assert tokens[i].tolist() == (seq if score > -math.inf else [-1] * len(steps))
