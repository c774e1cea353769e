"""Performance cases of the serving step's operators: what a program that serves a model has them do.

A case is a dict of plain values.  ``kind`` says which operator it is:

- ``tree``: ``co_alibi_decode_tree``, the step's new tokens (one token, a run of them or a tree of drafts)
  against a key / value cache and each other;
- ``append``: ``co_alibi_cache_append``, new keys and values written behind a cache's filled rows;
- ``sample``: ``co_alibi_sample``, the next tokens from logits and given uniform numbers.

``page`` is the rows per page of a paged cache, or 0 for one contiguous cache per sequence.  With
``ragged`` every sequence has a length of its own between 0 and ``L``, the longest ``L``; the lengths follow
from the case alone, so that its work does.

With ``own`` false ``run`` computes the operators from elementary torch operations; with it true it calls the
package.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _tree(name, B, Hq, Hkv, T, L, D, dtype, page, parents="tree", ragged=False, scale=0.5, lse=False):
    c = {"kind": "tree", "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "L": L, "D": D, "dtype": dtype, "page": page,
         "parents": parents, "ragged": ragged, "scale": scale, "lse": lse}
    return dict(c, name=name) if name else c


def _append(name, B, Hkv, T, L, D, dtype, page, mode="all", ragged=False, layout="bhsd"):
    c = {"kind": "append", "B": B, "Hkv": Hkv, "T": T, "L": L, "D": D, "dtype": dtype, "page": page, "mode": mode,
         "ragged": ragged, "layout": layout}
    return dict(c, name=name) if name else c


def _sample(name, B, V, dtype, temperature, top_k, top_p, min_p, per_row=False, masked=False, scale=2.5):
    c = {"kind": "sample", "B": B, "V": V, "dtype": dtype, "temperature": temperature, "top_k": top_k, "top_p": top_p,
         "min_p": min_p, "per_row": per_row, "masked": masked, "scale": scale}
    return dict(c, name=name) if name else c


def listed():
    return [
        # The next token of one short sequence of the 12-head GPT: latency counts.
        _tree("tree_token", 1, 12, 12, 1, 500, 64, "bf16", 64, parents="chain"),
        # fp32 validation of the same heads: the last 7 tokens of two prompts, over contiguous caches.
        _tree("tree_fp32", 2, 12, 12, 7, 1000, 64, "fp32", 0, parents="chain", lse=True),
        # One request of the grouped-query model, 16 drafted tokens after a long prompt.
        _tree("tree_gqa", 1, 32, 8, 16, 8192, 128, "bf16", 16),
        # 16 requests of different lengths, 24 drafts each.
        _tree("tree_serving", 16, 32, 8, 24, 8192, 128, "bf16", 64, ragged=True),
        # One very long context, the most drafts a step takes.
        _tree("tree_long", 1, 32, 8, 64, 131072, 128, "fp16", 256),
        # The key and value of one token for each of 16 requests.
        _append("append_token", 16, 8, 1, 1000, 128, "bf16", 64, ragged=True, layout="bshd"),
        # The accepted path of 24 drafts for each of 16 requests.
        _append("append_path", 16, 8, 24, 1000, 128, "bf16", 16, mode="path", ragged=True),
        # Eight prompts of different lengths, from a padded batch.
        _append("append_prompt", 8, 8, 2048, 0, 128, "bf16", 64, mode="counts", layout="bshd"),
        # One token of the GPT's vocabulary, fp32 logits.
        _sample("sample_one", 1, 50304, "fp32", 0.8, 50, 1.0, 0.0),
        # A serving batch, every request with its own settings.
        _sample("sample_serving", 64, 50304, "bf16", 0.9, 0, 0.95, 0.0, per_row=True),
        # Many samples over a large vocabulary, part of it forbidden by a grammar.
        _sample("sample_large", 256, 131071, "fp32", 1.0, 0, 0.9, 0.02, masked=True),
    ]


# ------------------------------------------------------------------ drawn cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(("tree", "append", "sample"), (5, 2, 3))[0]
    page = rng.choice((0, 16, 32, 64, 64, 128, 256))
    D = rng.choices((16, 32, 64, 128, 256), (1, 2, 4, 6, 1))[0]
    if kind == "tree":
        while True:
            hkv = rng.choice((1, 2, 4, 6, 8, 12, 16))
            hq = hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 4, 8) if g * hkv <= 32])
            dtype = rng.choices(("bf16", "fp16", "fp32"), (5, 3, 1))[0]
            c = _tree(None, _log_int(rng, 1, 48), hq, hkv, rng.choice((1, _log_int(rng, 1, 64), rng.randrange(2, 65))),
                      _log_int(rng, 1, 131072), D, dtype, page, rng.choice(("chain", "tree", "tree")), rng.random() < 0.6,
                      rng.choice((0.3, 0.5, 1.0)), rng.random() < 0.3)
            scores = c["B"] * hq * c["T"] * c["L"] * (8 if dtype == "fp32" else 1)
            if not (dtype == "fp32" and D == 256) and scores <= 1 << 28 and c["B"] * hkv * c["L"] * D <= 1 << 27:
                return c
    if kind == "append":
        while True:
            mode = rng.choice(("all", "counts", "path"))
            T = rng.randrange(1, 65) if mode == "path" else rng.choice((1, _log_int(rng, 1, 4096)))
            c = _append(None, _log_int(rng, 1, 64), rng.choice((1, 2, 4, 8, 12)), T, rng.choice((0, _log_int(rng, 1, 4096))),
                        D, rng.choice(("bf16", "fp16", "fp32")), page, mode, rng.random() < 0.6,
                        rng.choice(("bhsd", "bshd")))
            if c["B"] * c["Hkv"] * D * c["T"] <= 1 << 24 and c["B"] * c["Hkv"] * D * (c["T"] + c["L"]) <= 1 << 25:
                return c
    B = _log_int(rng, 1, 256)
    V = _log_int(rng, 100, 131072)
    return _sample(None, B, V, rng.choice(("fp32", "bf16", "fp16")), rng.choice((0.0, 0.6, 0.8, 1.0, 1.3)),
                   rng.choice((0, 0, 1, 40, rng.randrange(1, V + 1))), rng.choice((1.0, 1.0, 0.95, 0.9, 0.5)),
                   rng.choice((0.0, 0.0, 0.02, 0.1)), rng.random() < 0.4, rng.random() < 0.3, rng.choice((1.0, 2.5, 4.0)))


# ------------------------------------------------------------------ inputs


def _lens(c):
    """The filled rows of every sequence's cache."""
    if not c["ragged"]:
        return [c["L"]] * c["B"]
    rng = random.Random(1000003 * c["B"] + c["L"])
    lens = [rng.randrange(0, c["L"] + 1) for _ in range(c["B"])]
    lens[rng.randrange(c["B"])] = c["L"]
    return lens


def _counts(c):
    """The rows every sequence appends."""
    if c["mode"] == "all":
        return [c["T"]] * c["B"]
    rng = random.Random(1000033 * c["B"] + c["T"])
    most = c["T"] if c["mode"] == "counts" else min(c["T"], 8)
    return [rng.randrange(0, most + 1) for _ in range(c["B"])]


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _heads(gen, c, H, S, dtype, scale, bshd):
    """(B, H, S, D), as a projection leaves it (a transposed view) with bshd."""
    if bshd:
        return _normal(gen, (c["B"], S, H, c["D"]), dtype, scale).transpose(1, 2)
    return _normal(gen, (c["B"], H, S, c["D"]), dtype, scale)


def _cache(gen, c, rows, scale):
    """One cache of `rows` rows per sequence, and one unit (a page, or a sequence) more behind it that no
    sequence owns."""
    dt = DTYPES[c["dtype"]]
    if c["page"] == 0:
        return _normal(gen, (c["B"] + 1, c["Hkv"], rows, c["D"]), dt, scale)
    pages = c["B"] * -(-rows // c["page"])
    return _normal(gen, (pages + 1, c["Hkv"], c["page"], c["D"]), dt, scale)


def _table(gen, c, rows):
    """The block table: every sequence's pages, scattered over the pool."""
    if c["page"] == 0:
        return None
    n = -(-rows // c["page"])
    order = torch.randperm(c["B"] * n, generator=gen, device="cuda")
    return order.view(c["B"], n).to(torch.int32)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "sample":
        B, V = c["B"], c["V"]
        x = torch.randn((B, V), generator=gen, device="cuda") * c["scale"]
        if c["masked"]:
            x = x.masked_fill_(torch.rand((B, V), generator=gen, device="cuda") < 0.2, -math.inf)
        s["logits"] = x.to(dt)
        s["uniforms"] = torch.rand((B,), generator=gen, device="cuda")
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = c["temperature"], c["top_k"], c["top_p"], c["min_p"]
        if c["per_row"]:
            s["temperature"] = c["temperature"] * (0.5 + torch.rand((B,), generator=gen, device="cuda"))
            s["top_k"] = torch.randint(0, 200, (B,), generator=gen, device="cuda", dtype=torch.int32)
            s["top_p"] = 0.5 + 0.5 * torch.rand((B,), generator=gen, device="cuda")
            s["min_p"] = 0.1 * torch.rand((B,), generator=gen, device="cuda")
        return s
    B, T = c["B"], c["T"]
    s["seq_lens"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
    if c["kind"] == "append":
        cap = c["L"] + T + 3
        s["k"] = _heads(gen, c, c["Hkv"], T, dt, 1.0, c["layout"] == "bshd")
        s["v"] = _heads(gen, c, c["Hkv"], T, dt, 1.0, c["layout"] == "bshd")
        s["k_pool"], s["v_pool"] = _cache(gen, c, cap, 1.0), _cache(gen, c, cap, 1.0)
        s["table"] = _table(gen, c, cap)
        s["counts"] = None if c["mode"] == "all" else torch.tensor(_counts(c), dtype=torch.int32, device="cuda")
        s["rows"] = None
        if c["mode"] == "path":  # increasing rows of the new tokens, of which the first `counts` are taken
            n = min(T, 8)
            s["rows"] = torch.rand((B, T), generator=gen, device="cuda").argsort(1)[:, :n].sort(1).values.to(torch.int32)
        return s
    s["q"] = _heads(gen, c, c["Hq"], T, dt, c["scale"], True)
    s["k"] = _heads(gen, c, c["Hkv"], T, dt, c["scale"], True)
    s["v"] = _heads(gen, c, c["Hkv"], T, dt, c["scale"], True)
    cap = c["L"] + T
    s["k_pool"], s["v_pool"] = _cache(gen, c, cap, c["scale"]), _cache(gen, c, cap, c["scale"])
    s["table"] = _table(gen, c, cap)
    s["parents"] = None
    if c["parents"] == "tree":  # each draft hangs on one of the last few before it, or on the cache
        back = torch.randint(1, 7, (B, T), generator=gen, device="cuda")
        s["parents"] = (torch.arange(T, device="cuda") - back).clamp_(min=-1).to(torch.int32)
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "append": _plain_append, "sample": _plain_sample}[state["case"]["kind"]](state)


def _run_own(s):
    import co_alibi_attn as co

    c = s["case"]
    if c["kind"] == "sample":
        return co.co_alibi_sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"])
    k_cache, v_cache = s["k_pool"][:-1], s["v_pool"][:-1]
    if c["kind"] == "append":
        co.co_alibi_cache_append(s["k"], s["v"], k_cache, v_cache, s["seq_lens"], block_table=s["table"], rows=s["rows"],
                                 counts=s["counts"])
        return {"k_cache": k_cache, "v_cache": v_cache}
    out = co.co_alibi_decode_tree(s["q"], s["k"], s["v"], k_cache, v_cache, seq_len=s["seq_lens"], parents=s["parents"],
                                  block_table=s["table"], max_seq_len=c["L"], return_lse=c["lse"])
    return {"o": out[0], "lse": out[1]} if c["lse"] else out


def _plain_slopes(heads, dtype):
    """Penalty slope of every query head, rounded to the inputs' type."""
    n = 1 << (heads.bit_length() - 1)
    s = torch.pow(2.0 ** (-8.0 / n), torch.arange(1, n + 1))
    if heads > n:
        s = torch.cat([s, torch.pow(2.0 ** (-4.0 / n), torch.arange(1, 2 * (heads - n), 2))])
    return (2.0 * s).to(dtype).float().cuda()


def _filled(pool, table, rows):
    """(B, Hkv, rows, D): the sequences' caches, their pages put in order."""
    if table is None:
        return pool[:-1, :, :rows]
    B, n = table.shape
    _, H, page, D = pool.shape
    return pool[table.long()].transpose(1, 2).reshape(B, H, n * page, D)[:, :, :rows]


def _plain_tree(s):
    c = s["case"]
    B, Hq, Hkv, T, L, D = c["B"], c["Hq"], c["Hkv"], c["T"], c["L"], c["D"]
    G = Hq // Hkv
    dt = s["q"].dtype
    node = torch.arange(T, device="cuda")
    if s["parents"] is None:
        sees = (node[None, :] <= node[:, None]).expand(B, T, T)
    else:
        # A node sees itself and what its parent sees.
        eye = torch.eye(T, dtype=torch.bool, device="cuda")
        known = [eye[0].expand(B, T)]
        for t in range(1, T):
            par = s["parents"][:, t].long()
            above = torch.stack(known, 1)[torch.arange(B, device="cuda"), par.clamp(min=0)]
            known.append((above & (par >= 0)[:, None]) | eye[t])
        sees = torch.stack(known, 1)
    filled = torch.arange(L, device="cuda")[None, :] < s["seq_lens"][:, None]
    ok = torch.cat([filled[:, None, :].expand(B, T, L), sees], 2)  # (B, T, L + T)
    ok = ok[:, None, None]
    keys = torch.cat([_filled(s["k_pool"], s["table"], L), s["k"]], 2).float()
    vals = torch.cat([_filled(s["v_pool"], s["table"], L), s["v"]], 2).float()
    # Unfilled rows may hold anything.
    vals[:, :, :L].masked_fill_(~filled[:, None, :, None], 0.0)
    q = s["q"].float().reshape(B, Hkv, G * T, D)
    t = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, Hkv, G, T, L + T)
    t = torch.where(ok, t, -math.inf)
    z = torch.sigmoid(t).flip(4).cumsum(4, dtype=torch.float64).flip(4)
    a = t - _plain_slopes(Hq, dt).view(1, Hkv, G, 1, 1) * z
    del t, z
    m = a.amax(4, keepdim=True)
    p = torch.exp((a - m).float())
    l = p.sum(4, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, G * T, L + T), vals).view(B, Hkv, G, T, D) / l
    o = o.view(B, Hq, T, D).to(dt)
    if not c["lse"]:
        return o
    return {"o": o, "lse": (m + torch.log(l)).float().view(B, Hq, T)}


def _plain_append(s):
    c = s["case"]
    B, T, page = c["B"], c["T"], c["page"]
    rows = torch.arange(T, device="cuda").expand(B, T) if s["rows"] is None else s["rows"].long()
    n = rows.shape[1]
    i = torch.arange(n, device="cuda")
    pos = s["seq_lens"][:, None] + i
    seq = torch.arange(B, device="cuda")[:, None].expand(B, n)
    ok = torch.ones_like(rows, dtype=torch.bool) if s["counts"] is None else i < s["counts"][:, None]
    if page == 0:
        unit, off, spare = seq, pos, B
    else:
        unit, off, spare = s["table"][seq, pos // page].long(), pos % page, s["k_pool"].shape[0] - 1
    # Rows past a sequence's count go to the unit that no sequence owns.
    unit = torch.where(ok, unit, spare)
    off = torch.where(ok, off, 0)
    for name in ("k", "v"):
        s[name + "_pool"][unit, :, off] = s[name].transpose(1, 2)[seq, rows]
    return {"k_cache": s["k_pool"][:-1], "v_cache": s["v_pool"][:-1]}


def _column(x, B, dtype):
    """A setting as one value per row."""
    return x.to(dtype)[:, None] if torch.is_tensor(x) else torch.full((B, 1), x, dtype=dtype, device="cuda")


def _plain_sample(s):
    x = s["logits"].float()
    B, V = x.shape
    temp = _column(s["temperature"], B, torch.float64)
    top_k = _column(s["top_k"], B, torch.int64)
    top_p, min_p = _column(s["top_p"], B, torch.float64), _column(s["min_p"], B, torch.float64)
    vals, idx = torch.sort(x, dim=1, descending=True, stable=True)
    top = vals[:, :1].double()
    greedy = temp <= 0
    w = torch.where(vals == vals[:, :1], 1.0, torch.exp((vals.double() - top) / torch.where(greedy, 1.0, temp)))
    rank = torch.arange(V, device="cuda")
    w = torch.where((rank < top_k) | (top_k <= 0), w, 0.0)
    mass = w.cumsum(1)
    keep = ((mass - w < top_p * mass[:, -1:]) | (top_p >= 1)) & (w >= min_p) & (w > 0)
    keep[:, 0] = True
    kept = (w * keep).cumsum(1)
    past = (kept <= s["uniforms"].double()[:, None] * kept[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(past, keep.sum(1, keepdim=True) - 1)
    token = idx.gather(1, torch.where(greedy, 0, at))[:, 0]
    bad = torch.isnan(x).any(1) | (top[:, 0] == -math.inf)
    return torch.where(bad, -1, token)


# ------------------------------------------------------------------ the work a pass cannot do without


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "sample":
        # Each logit is read, scaled, and its exponential added up; a comparison for the order.
        return {"bytes": c["B"] * (c["V"] * size + 4 + 8), "flops": 4 * c["B"] * c["V"]}
    if c["kind"] == "append":
        rows = sum(_counts(c)) * c["Hkv"] * c["D"]
        return {"bytes": 4 * size * rows + 4 * c["B"], "flops": 0}
    new = c["B"] * c["T"] * c["D"]
    rows = sum(_lens(c))
    return {"bytes": size * (2 * rows * c["Hkv"] * c["D"] + 2 * new * c["Hkv"] + 2 * new * c["Hq"]),
            "flops": 4 * c["D"] * c["Hq"] * c["T"] * (rows + c["B"])}


# ------------------------------------------------------------------ the results in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "append": _exact_append, "sample": _exact_sample}[case["kind"]](s)


def _exact_tree(s):
    """Every node by itself: its keys are the filled rows, then the path from the root to the node."""
    c = s["case"]
    B, Hq, Hkv, T, D = c["B"], c["Hq"], c["Hkv"], c["T"], c["D"]
    G = Hq // Hkv
    n = 2 ** int(math.log2(Hq))
    lam = [2.0 * 2.0 ** (-8.0 * (h + 1) / n) for h in range(n)]
    lam += [2.0 * 2.0 ** (-4.0 * (2 * h + 1) / n) for h in range(Hq - n)]
    lam = torch.tensor(lam, dtype=torch.float32, device="cuda").to(DTYPES[c["dtype"]]).double().view(Hkv, G, 1)
    o = torch.zeros((B, Hq, T, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, Hq, T), dtype=torch.float64, device="cuda")
    parents = [list(range(-1, T - 1))] * B if s["parents"] is None else s["parents"].tolist()
    lens = _lens(c)
    for b in range(B):
        if c["page"] == 0:
            kc, vc = (s[x][b, :, :lens[b]].double() for x in ("k_pool", "v_pool"))
        else:
            own_pages = s["table"][b].tolist()[:-(-lens[b] // c["page"])]
            kc, vc = (torch.cat([s[x][i] for i in own_pages] or [s[x][0]], 1)[:, :lens[b]].double()
                      for x in ("k_pool", "v_pool"))
        q, k, v = (s[x][b].double() for x in ("q", "k", "v"))
        q = q.reshape(Hkv, G, T, D)
        kct = kc.transpose(1, 2).contiguous()
        for t in range(T):
            path = [t]
            while parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            qt = q[:, :, t]
            x = torch.cat([qt @ kct, qt @ k[:, path].transpose(1, 2).contiguous()], 2) / math.sqrt(D)
            sig = 1.0 / (1.0 + torch.exp(-x))
            x = x - lam * (sig.sum(2, keepdim=True) - sig.cumsum(2) + sig)
            top = x.max(2, keepdim=True).values
            e = torch.exp(x - top)
            den = e.sum(2, keepdim=True)
            o[b, :, t] = ((e[:, :, :lens[b]] @ vc + e[:, :, lens[b]:] @ v[:, path]) / den).reshape(Hq, D)
            lse[b, :, t] = (top + torch.log(den)).reshape(Hq)
    return {"o": o, "lse": lse} if c["lse"] else o


def _exact_append(s):
    c = s["case"]
    lens, counts, page = _lens(c), _counts(c), c["page"]
    out = {}
    for name in ("k", "v"):
        new = s[name].double().cpu()
        cache = s[name + "_pool"][:-1].double().cpu()
        for b in range(c["B"]):
            for i in range(counts[b]):
                row = i if s["rows"] is None else int(s["rows"][b, i])
                at = lens[b] + i
                if page == 0:
                    cache[b, :, at] = new[b, :, row]
                else:
                    cache[int(s["table"][b, at // page]), :, at % page] = new[b, :, row]
        out[name + "_cache"] = cache.cuda()
    return out


def _exact_sample(s):
    import numpy as np

    c = s["case"]
    x = s["logits"].double().cpu().numpy()
    u = s["uniforms"].double().cpu().numpy()

    def setting(name, b):
        return s[name][b].item() if torch.is_tensor(s[name]) else s[name]

    out = []
    for b in range(c["B"]):
        order = np.argsort(-x[b], kind="stable")
        temp, k, p, m = (setting(name, b) for name in ("temperature", "top_k", "top_p", "min_p"))
        if temp <= 0:
            out.append(int(order[0]))
            continue
        if k > 0:
            order = order[:k]
        w = np.exp((x[b][order] - x[b][order[0]]) / temp)
        before = np.concatenate([[0.0], np.cumsum(w)])
        if p < 1:
            n = max(1, int(np.searchsorted(before[:-1], p * before[-1], side="left")))
            w = w[:n]
        w = w[(w >= m) & (w > 0)]
        cum = np.cumsum(w)
        out.append(int(order[min(int(np.searchsorted(cum, u[b] * cum[-1], side="right")), len(w) - 1)]))
    return torch.tensor(out, device="cuda")
