"""Performance cases of an 8-bit key / value cache and of beam search: what a program that serves a model has them do.

A case is a dict of plain values.  ``kind`` says which operator it is:

- ``tree``: ``co_alibi_decode_tree_8bit``, the step's new tokens against a cache held in 8 bits, and each other;
- ``append``: ``co_alibi_cache_append_8bit``, new keys and values quantised as they are written behind the filled rows;
- ``read``: ``co_alibi_cache_read_8bit``, rows of such a cache as ordinary keys and values;
- ``select``: ``co_alibi_beam_select``, the best continuations over the beams of a sequence and the vocabulary;
- ``reorder``: ``co_alibi_cache_reorder``, a paged cache whose sequences take over the rows of their parents.

An 8-bit cache holds a code per element (``format``: e4m3, or int8 in [-127, 127]) and a scale for each kv head's blocks of
16 rows; the value is their product.  A block's scale is the least power of two, from 2^-40 on, at which no code passes the
format's largest value (448, 127); rows added to a block that has some double the scale as often as they need, and the codes
it holds are halved as often (each rounding to the nearest code, ties to even).

``page`` is the rows per page of a paged cache, or 0 for one contiguous cache per sequence.  With ``ragged`` every sequence
has a length of its own between 0 and ``L``, the longest ``L``; the lengths follow from the case alone, so that its work does.

With ``own`` false ``run`` computes the operators from elementary torch operations; with it true it calls the package.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
RUN = 16  # rows of a block
LEAST = -40  # a scale's smallest exponent


def _tree(name, B, Hq, Hkv, T, L, D, dtype, fmt, page, parents="tree", ragged=False, scale=0.5, lse=False):
    c = {"kind": "tree", "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "L": L, "D": D, "dtype": dtype, "format": fmt, "page": page,
         "parents": parents, "ragged": ragged, "scale": scale, "lse": lse}
    return dict(c, name=name) if name else c


def _append(name, B, Hkv, T, L, D, dtype, fmt, page, mode="all", ragged=False, layout="bhsd"):
    c = {"kind": "append", "B": B, "Hkv": Hkv, "T": T, "L": L, "D": D, "dtype": dtype, "format": fmt, "page": page,
         "mode": mode, "ragged": ragged, "layout": layout}
    return dict(c, name=name) if name else c


def _read(name, B, Hkv, L, N, D, dtype, fmt, page, ragged=False, later=False):
    c = {"kind": "read", "B": B, "Hkv": Hkv, "L": L, "N": N, "D": D, "dtype": dtype, "format": fmt, "page": page,
         "ragged": ragged, "later": later}
    return dict(c, name=name) if name else c


def _select(name, B, W, N, V, dtype, done=False, masked=False, scale=2.5):
    c = {"kind": "select", "B": B, "W": W, "N": N, "V": V, "dtype": dtype, "done": done, "masked": masked, "scale": scale}
    return dict(c, name=name) if name else c


def _reorder(name, B, W, layers, Hkv, L, D, dtype, page, ragged=False, spread=1.0):
    c = {"kind": "reorder", "B": B, "W": W, "layers": layers, "Hkv": Hkv, "L": L, "D": D, "dtype": dtype, "page": page,
         "ragged": ragged, "spread": spread}
    return dict(c, name=name) if name else c


def listed():
    return [
        # The next token of one short sequence of the 12-head GPT: latency counts.
        _tree("tree8_token", 1, 12, 12, 1, 500, 64, "bf16", "e4m3", 64, parents="chain"),
        # The next token of 32 requests of different lengths of the grouped-query model: the cache's bytes count.
        _tree("tree8_serving", 32, 32, 8, 1, 8192, 128, "bf16", "e4m3", 64, parents="chain", ragged=True),
        # 16 requests, 24 drafts each: the products and exponentials count.
        _tree("tree8_drafts", 16, 32, 8, 24, 8192, 128, "bf16", "int8", 64, ragged=True),
        # One very long context, a few drafts, with the statistics that a merge with other keys needs.
        _tree("tree8_long", 1, 32, 8, 7, 131072, 128, "fp16", "e4m3", 256, lse=True),
        # The key and value of one token for each of 16 requests: blocks that are begun, filled up and rescaled.
        _append("append8_token", 16, 8, 1, 1000, 128, "bf16", "e4m3", 64, ragged=True, layout="bshd"),
        # Eight prompts of different lengths, from a padded batch.
        _append("append8_prompt", 8, 8, 2048, 0, 128, "bf16", "int8", 64, mode="counts", layout="bshd"),
        # One validation sequence of the GPT's heads, in fp32.
        _read("read8_one", 1, 12, 500, 500, 64, "fp32", "int8", 0),
        # Eight prompts' rows for a forward over whole sequences.
        _read("read8_prompts", 8, 8, 4096, 4096, 128, "bf16", "e4m3", 64, ragged=True),
        # Four beams of one sequence over the GPT's vocabulary, fp32 logits.
        _select("select_one", 1, 4, 4, 50304, "fp32"),
        # Eight beams of 16 sequences over a large vocabulary, some of them finished.
        _select("select_serving", 16, 8, 8, 131071, "bf16", done=True),
        # Four beams of the 12-layer GPT.
        _reorder("reorder_one", 1, 4, 12, 12, 777, 64, "bf16", 64),
        # Eight beams of 16 sequences of the grouped-query model, 8-bit pages of four layers.
        _reorder("reorder_serving", 16, 8, 4, 8, 1000, 128, "e4m3", 64, ragged=True),
    ]


# ------------------------------------------------------------------ drawn cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(("tree", "append", "read", "select", "reorder"), (5, 3, 2, 3, 2))[0]
    page = rng.choice((0, 16, 32, 64, 64, 128, 256))
    D = rng.choices((16, 32, 64, 128, 256), (1, 2, 4, 6, 1))[0]
    fmt = rng.choice(("e4m3", "int8"))
    if kind == "tree":
        while True:
            hkv = rng.choice((1, 2, 4, 6, 8, 12, 16))
            hq = hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 4, 8) if g * hkv <= 32])
            dtype = rng.choices(("bf16", "fp16", "fp32"), (5, 3, 1))[0]
            c = _tree(None, _log_int(rng, 1, 48), hq, hkv, rng.choice((1, 1, _log_int(rng, 1, 64), rng.randrange(2, 65))),
                      _log_int(rng, 1, 131072), D, dtype, fmt, page, rng.choice(("chain", "tree", "tree")),
                      rng.random() < 0.6, rng.choice((0.3, 0.5, 1.0)), rng.random() < 0.3)
            scores = c["B"] * hq * c["T"] * c["L"] * (8 if dtype == "fp32" else 1)
            if not (dtype == "fp32" and D == 256) and scores <= 3 << 25 and c["B"] * hkv * c["L"] * D <= 1 << 27:
                return c
    if kind == "append":
        while True:
            mode = rng.choice(("all", "counts", "path"))
            T = rng.randrange(1, 65) if mode == "path" else rng.choice((1, _log_int(rng, 1, 4096)))
            c = _append(None, _log_int(rng, 1, 64), rng.choice((1, 2, 4, 8, 12)), T, rng.choice((0, _log_int(rng, 1, 4096))),
                        D, rng.choice(("bf16", "fp16", "fp32")), fmt, page, mode, rng.random() < 0.6,
                        rng.choice(("bhsd", "bshd")))
            if c["B"] * c["Hkv"] * D * c["T"] <= 1 << 24 and c["B"] * c["Hkv"] * D * (c["T"] + c["L"]) <= 1 << 25:
                return c
    if kind == "read":
        while True:
            L = _log_int(rng, 1, 8192)
            c = _read(None, _log_int(rng, 1, 64), rng.choice((1, 2, 4, 8, 12)), L, rng.choice((L, rng.randrange(1, L + 1))),
                      D, rng.choice(("bf16", "fp16", "fp32")), fmt, page, rng.random() < 0.6, rng.random() < 0.4)
            if c["B"] * c["Hkv"] * D * L <= 1 << 25:
                return c
    if kind == "select":
        while True:
            W = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
            c = _select(None, _log_int(rng, 1, 32), W, rng.choice((W, W, W, rng.randrange(1, 33))), _log_int(rng, 100, 131072),
                        rng.choice(("fp32", "bf16", "fp16")), rng.random() < 0.4, rng.random() < 0.3,
                        rng.choice((1.0, 2.5, 4.0)))
            if c["B"] * W * c["V"] <= 1 << 24:
                return c
    while True:
        c = _reorder(None, _log_int(rng, 1, 32), rng.choice((1, 2, 3, 4, 5, 8, 16)), rng.choice((1, 2, 4, 12)),
                     rng.choice((1, 2, 4, 8, 12)), _log_int(rng, 1, 4096), D, rng.choice(("e4m3", "int8", "bf16", "fp32")),
                     page or 64, rng.random() < 0.6, rng.choice((0.3, 1.0, 3.0)))
        size = {"fp32": 4, "bf16": 2}.get(c["dtype"], 1)
        if c["B"] * c["W"] * c["layers"] * c["Hkv"] * (c["L"] + c["page"]) * D * size <= 1 << 29:
            return c


# ------------------------------------------------------------------ inputs


def _lens(c):
    """The filled rows of every sequence's cache (of every group of beams)."""
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


def _firsts(c):
    """The first row that is read of every sequence."""
    if not c["later"]:
        return [0] * c["B"]
    rng = random.Random(1000037 * c["B"] + c["L"])
    return [rng.randrange(0, c["L"] - c["N"] + 1) for _ in range(c["B"])]


def _parents(c):
    """The beam that every beam continues: the better ones, of lower places, more often with a small `spread`."""
    rng = random.Random(1000039 * c["B"] + 101 * c["W"] + c["L"])
    return [sorted(min(c["W"] - 1, int(c["W"] * rng.random() ** (1 / c["spread"]))) for _ in range(c["W"]))
            for _ in range(c["B"])]


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _heads(gen, c, H, S, dtype, scale, bshd):
    """(B, H, S, D), as a projection leaves it (a transposed view) with bshd."""
    if bshd:
        return _normal(gen, (c["B"], S, H, c["D"]), dtype, scale).transpose(1, 2)
    return _normal(gen, (c["B"], H, S, c["D"]), dtype, scale)


def _least_exponent(top, fmt):
    """The least k with top <= 2^k times the format's largest code."""
    m, e = torch.frexp(top)  # top = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9, 127 = 0.9921875 * 2^7
    k = e - 9 + (m > 0.875).int() if fmt == "e4m3" else e - 7 + (m > 0.9921875).int()
    return torch.where(top > 0, k, LEAST).clamp(min=LEAST)


def _two_to(k):
    """2^k in fp32, exactly."""
    return (k.int() + 127 << 23).view(torch.float32)


def _code(x, fmt):
    """The nearest codes of x, as fp32 values."""
    return x.to(torch.float8_e4m3fn).float() if fmt == "e4m3" else torch.round(x)


def _cache8(gen, c, rows, scale):
    """Codes and scales of one cache of `rows` rows per sequence, and one unit (a page, or a sequence) more behind it that no
    sequence owns.  The blocks differ in size, as the keys and values of a text do."""
    units = c["B"] + 1 if c["page"] == 0 else c["B"] * -(-rows // c["page"]) + 1
    n = rows if c["page"] == 0 else c["page"]
    blocks = -(-n // RUN)
    codes = torch.empty((units, c["Hkv"], n, c["D"]), dtype=CODES[c["format"]], device="cuda")
    scales = torch.empty((units, c["Hkv"], blocks), device="cuda")
    step = max(1, (1 << 26) // (c["Hkv"] * blocks * RUN * c["D"]))
    for i in range(0, units, step):
        u = min(units, i + step) - i
        x = torch.randn((u, c["Hkv"], blocks, RUN, c["D"]), generator=gen, device="cuda")
        x *= scale * torch.exp2(0.5 * torch.randn((u, c["Hkv"], blocks, 1, 1), generator=gen, device="cuda"))
        s = _two_to(_least_exponent(x.abs().amax((3, 4)), c["format"]))
        scales[i:i + u] = s
        x = (x / s[..., None, None]).view(u, c["Hkv"], blocks * RUN, c["D"])[:, :, :n]
        codes[i:i + u] = (x if c["format"] == "e4m3" else torch.round(x)).to(codes.dtype)
    return codes, scales


def _table(gen, c, rows):
    """The block table: every sequence's pages, scattered over the pool."""
    if c["page"] == 0:
        return None
    n = -(-rows // c["page"])
    order = torch.randperm(c["B"] * n, generator=gen, device="cuda")
    return order.view(c["B"], n).to(torch.int32)


def _prepare_select(c, gen, s):
    B, W, V = c["B"], c["W"], c["V"]
    x = torch.randn((B, W, V), generator=gen, device="cuda") * c["scale"]
    if c["masked"]:
        x = x.masked_fill_(torch.rand((B, W, V), generator=gen, device="cuda") < 0.2, -math.inf)
    s["logits"] = x.to(DTYPES[c["dtype"]])
    s["scores"] = -20 * torch.rand((B, W), generator=gen, device="cuda").sort(1).values
    s["finished"] = torch.rand((B, W), generator=gen, device="cuda") < 0.3 if c["done"] else None


def _prepare_reorder(c, gen, s):
    """Beams some steps behind the prompt: they share its pages and hold, or share, pages of their own behind it."""
    B, W, page = c["B"], c["W"], c["page"]
    blocks = -(-(c["L"] + 8) // page)
    pages = torch.randperm(B * W * blocks, generator=gen, device="cuda").view(B, W, blocks)
    lens = torch.tensor(_lens(c), device="cuda")
    held = torch.arange(W, device="cuda")[None, :, None].expand(B, W, blocks).clone()
    column = torch.arange(blocks, device="cuda")
    full = (column + 1) * page <= lens[:, None]  # (B, blocks)
    shared = torch.randint(0, W, (B, W, blocks), generator=gen, device="cuda")
    shared = torch.where((column < blocks // 2)[None, None], 0, shared)
    held = torch.where(full[:, None], shared, held)
    s["pages"] = pages.view(B * W, blocks).to(torch.int32)
    s["table"] = pages.gather(1, held).view(B * W, blocks).to(torch.int32)
    s["lens"] = lens.repeat_interleave(W).to(torch.int32)
    s["parents"] = torch.tensor(_parents(c), dtype=torch.int32, device="cuda")
    s["pools"] = []
    shape = (B * W * blocks, c["Hkv"], page, c["D"])
    eight = c["dtype"] in CODES
    for _ in range(2 * c["layers"]):
        if eight:
            x = torch.randint(0, 255, shape, generator=gen, device="cuda", dtype=torch.uint8)
            x = torch.where((x & 127) == 127, 0, x)  # (no NaN among the e4m3 codes)
            s["pools"].append(x.view(CODES[c["dtype"]]))
        else:
            s["pools"].append(torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[c["dtype"]]))
    if eight:
        s["pools"] += [torch.rand((shape[0], c["Hkv"], page // RUN), generator=gen, device="cuda") for _ in s["pools"]]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "select":
        _prepare_select(c, gen, s)
        return s
    if c["kind"] == "reorder":
        _prepare_reorder(c, gen, s)
        return s
    dt = DTYPES[c["dtype"]]
    s["seq_lens"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
    T = c.get("T", 0)
    cap = c["L"] + T + 3
    scale = c.get("scale", 1.0)
    s["k_codes"], s["k_scale"] = _cache8(gen, c, cap, scale)
    s["v_codes"], s["v_scale"] = _cache8(gen, c, cap, scale)
    s["table"] = _table(gen, c, cap)
    if c["kind"] == "read":
        s["first"] = torch.tensor(_firsts(c), dtype=torch.int32, device="cuda") if c["later"] else None
        return s
    bshd = c["kind"] == "tree" or c["layout"] == "bshd"
    s["k"] = _heads(gen, c, c["Hkv"], T, dt, scale, bshd)
    s["v"] = _heads(gen, c, c["Hkv"], T, dt, scale, bshd)
    if c["kind"] == "append":
        s["counts"] = None if c["mode"] == "all" else torch.tensor(_counts(c), dtype=torch.int32, device="cuda")
        s["rows"] = None
        if c["mode"] == "path":  # increasing rows of the new tokens, of which the first `counts` are taken
            n = min(T, 8)
            s["rows"] = torch.rand((c["B"], T), generator=gen, device="cuda").argsort(1)[:, :n].sort(1).values.to(torch.int32)
        return s
    s["q"] = _heads(gen, c, c["Hq"], T, dt, scale, True)
    s["parents"] = None
    if c["parents"] == "tree":  # each draft hangs on one of the last few before it, or on the cache
        back = torch.randint(1, 7, (c["B"], T), generator=gen, device="cuda")
        s["parents"] = (torch.arange(T, device="cuda") - back).clamp_(min=-1).to(torch.int32)
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "append": _plain_append, "read": _plain_read, "select": _plain_select,
            "reorder": _plain_reorder}[state["case"]["kind"]](state)


def _run_own(s):
    import co_alibi_attn as co

    c = s["case"]
    if c["kind"] == "select":
        scores, parents, tokens = co.co_alibi_beam_select(s["logits"], s["scores"], num_beams=c["N"], finished=s["finished"],
                                                          end_token=2)
        return {"scores": scores, "parents": parents, "tokens": tokens}
    if c["kind"] == "reorder":
        table, lens = co.co_alibi_cache_reorder(s["pools"], s["lens"], s["parents"], s["table"], s["pages"])
        return {"table": table, "lens": lens, "pools": s["pools"]}
    cache = [s[x][:-1] for x in ("k_codes", "v_codes", "k_scale", "v_scale")]
    if c["kind"] == "read":
        k, v = co.co_alibi_cache_read_8bit(*cache, s["seq_lens"], c["N"], dtype=DTYPES[c["dtype"]], block_table=s["table"],
                                           first=s["first"])
        return {"k": k, "v": v}
    if c["kind"] == "append":
        co.co_alibi_cache_append_8bit(s["k"], s["v"], *cache, s["seq_lens"], block_table=s["table"], rows=s["rows"],
                                      counts=s["counts"])
        return dict(zip(("k_codes", "v_codes", "k_scale", "v_scale"), cache))
    out = co.co_alibi_decode_tree_8bit(s["q"], s["k"], s["v"], *cache, seq_len=s["seq_lens"], parents=s["parents"],
                                       block_table=s["table"], max_seq_len=c["L"], return_lse=c["lse"])
    return {"o": out[0], "lse": out[1]} if c["lse"] else out


def _plain_slopes(heads, dtype):
    """Penalty slope of every query head, rounded to the inputs' type."""
    n = 1 << (heads.bit_length() - 1)
    s = torch.pow(2.0 ** (-8.0 / n), torch.arange(1, n + 1))
    if heads > n:
        s = torch.cat([s, torch.pow(2.0 ** (-4.0 / n), torch.arange(1, 2 * (heads - n), 2))])
    return (2.0 * s).to(dtype).float().cuda()


def _place(s, pos):
    """The unit and the row in it of every cache row pos (B, n)."""
    c = s["case"]
    seq = torch.arange(c["B"], device="cuda")[:, None].expand_as(pos)
    if c["page"] == 0:
        return seq, pos.clamp(max=s["k_codes"].shape[2] - 1)
    at = (pos // c["page"]).clamp(max=s["table"].shape[1] - 1)
    return s["table"][seq, at].long(), pos % c["page"]


def _values(s, name, pos):
    """(B, Hkv, n, D) in fp32: the cache rows pos (B, n)."""
    unit, row = _place(s, pos)
    codes = s[name + "_codes"].view(torch.uint8)[unit, :, row].view(CODES[s["case"]["format"]]).float()
    return (codes * s[name + "_scale"][unit, :, row // RUN][..., None]).transpose(1, 2)


def _plain_tree(s):
    c = s["case"]
    B, Hq, Hkv, T, L, D = c["B"], c["Hq"], c["Hkv"], c["T"], c["L"], c["D"]
    G = Hq // Hkv
    dt = s["q"].dtype
    node = torch.arange(T, device="cuda")
    sees = (node[None, :] <= node[:, None]).expand(B, T, T)
    if s["parents"] is not None:
        # A node sees itself and what is up to T - 1 parents away.
        par = s["parents"].long()
        up = torch.eye(T, device="cuda") + (node == par[:, :, None]).float()
        sees = torch.linalg.matrix_power(up, max(T - 1, 1)) > 0
    row = torch.arange(L, device="cuda").expand(B, L)
    filled = row < s["seq_lens"][:, None]
    ok = torch.cat([filled[:, None, :].expand(B, T, L), sees], 2)[:, None, None]  # (B, 1, 1, T, L + T)
    keys = torch.cat([_values(s, "k", row), s["k"].float()], 2)
    vals = torch.cat([_values(s, "v", row), s["v"].float()], 2)
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
    B, T, H, D, fmt = c["B"], c["T"], c["Hkv"], c["D"], c["format"]
    rows = torch.arange(T, device="cuda").expand(B, T) if s["rows"] is None else s["rows"].long()
    n = rows.shape[1]
    lens = s["seq_lens"].long()[:, None]
    counts = torch.full((B, 1), n, device="cuda") if s["counts"] is None else s["counts"].long()[:, None]
    # Every sequence's blocks that may get rows, from the one of its next row on.
    nb = -(-(n + RUN - 1) // RUN)
    pos = lens // RUN * RUN + torch.arange(nb * RUN, device="cuda")
    old, new = pos < lens, (pos >= lens) & (pos < lens + counts)
    touched = new.view(B, nb, RUN).any(2)
    seq = torch.arange(B, device="cuda")[:, None]
    unit, row = _place(s, pos)
    spare = s["k_codes"].shape[0] - 1
    # Blocks without a new row go to the unit that no sequence owns.
    gets = (new | old) & touched.repeat_interleave(RUN, 1)
    unit_to, row_to = torch.where(gets, unit, spare), torch.where(gets, row, 0)
    block_unit = torch.where(touched, unit[:, ::RUN], spare)
    block = torch.where(touched, row[:, ::RUN] // RUN, 0)
    source = rows.gather(1, (pos - lens).clamp(0, n - 1))
    out = {}
    for name in ("k", "v"):
        codes, scales = s[name + "_codes"], s[name + "_scale"]
        x = s[name].transpose(1, 2)[seq, source].float()  # (B, rows, H, D)
        x = torch.where(new[..., None, None], x, 0.0).view(B, nb, RUN, H, D)
        top = x.abs().amax((2, 4))  # (B, nb, H)
        had = old.view(B, nb, RUN)[:, :, 0, None]
        fresh = _least_exponent(top, fmt)
        was = scales[block_unit, :, block]
        # The scale of a block that has rows: doubled as often as the new ones need it.
        held = torch.frexp(was).exponent - 1
        k = torch.where(had, torch.maximum(held, fresh), fresh)
        scale = _two_to(k)
        cells = codes.view(torch.uint8)[unit, :, row].view(codes.dtype).float().view(B, nb, RUN, H, D)
        shrunk = cells * torch.where(had, _two_to(held - k), 1.0)[:, :, None, :, None]
        x = _code(torch.where(new.view(B, nb, RUN)[..., None, None], x / scale[:, :, None, :, None], shrunk), fmt)
        codes.view(torch.uint8)[unit_to, :, row_to] = x.view(B, nb * RUN, H, D).to(codes.dtype).view(torch.uint8)
        scales[block_unit, :, block] = scale
        # The codes are what the values are held in: whole numbers, or e4m3's own values; times the scales they are the cache's.
        out[name + "_codes"], out[name + "_scale"] = codes[:-1], scales[:-1]
    return out


def _plain_read(s):
    c = s["case"]
    pos = torch.arange(c["N"], device="cuda").expand(c["B"], c["N"])
    if s["first"] is not None:
        pos = pos + s["first"].long()[:, None]
    filled = (pos < s["seq_lens"][:, None])[:, None, :, None]
    return {x: torch.where(filled, _values(s, x, pos), 0.0).to(DTYPES[c["dtype"]]) for x in ("k", "v")}


def _plain_select(s):
    c = s["case"]
    B, W, V, N = c["B"], c["W"], c["V"], c["N"]
    x = s["logits"].double()
    top = x.amax(2, keepdim=True)
    x = x - top
    x = x - torch.log(torch.exp(x).sum(2, keepdim=True)) + s["scores"].double()[:, :, None]
    if s["finished"] is not None:
        only = torch.where(torch.arange(V, device="cuda") == 2, s["scores"].double()[:, :, None], -math.inf)
        x = torch.where(s["finished"][:, :, None], only, x)
    best, at = torch.sort(x.view(B, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :N], at[:, :N]
    none = best == -math.inf
    return {"scores": best.float(), "parents": torch.where(none, 0, at // V).int(), "tokens": torch.where(none, -1, at % V)}


def _plain_reorder(s):
    c = s["case"]
    B, W, page = c["B"], c["W"], c["page"]
    J = s["table"].shape[1]
    par = s["parents"].long()
    group = torch.arange(B, device="cuda")[:, None]
    home = s["pages"].long().view(B, W, J)
    lens = s["lens"].long().view(B, W).gather(1, par)
    held = s["table"].long().view(B, W, J)[group, par]  # the parents' pages
    column = torch.arange(J, device="cuda")
    filled = (lens[:, :, None] - column * page).clamp(0, page)
    full, part = filled == page, (filled > 0) & (filled < page)
    # A page that is not full is its beam's alone: of those that want one, the first keeps it if no other beam has it full.
    same = held[:, :, None] == held[:, None]  # (B, W, W, J)
    before = torch.arange(W, device="cuda")[:, None] > torch.arange(W, device="cuda")
    taken = (same & (full[:, None] | (part[:, None] & before[None, :, :, None]))).any(2)
    keeps = full | (part & ~taken)
    # The others get, in order, the pages of the column that nobody keeps.
    used = ((home[:, :, None] == held[:, None]) & keeps[:, None]).any(2)  # (B, W, J)
    free = home.gather(1, used.int().sort(dim=1, stable=True).indices)
    place = ((~keeps).int().cumsum(1) - 1).clamp(min=0)
    now = torch.where(keeps, held, free.gather(1, place))
    # The copy of every beam's page that is not full (onto itself where it is kept).
    at = (lens // page).clamp(max=J - 1)[:, :, None]
    moves = (part & ~keeps).gather(2, at)
    to = now.gather(2, at).reshape(-1)
    of = torch.where(moves, held.gather(2, at), now.gather(2, at)).reshape(-1)
    rows = filled.gather(2, at).reshape(-1)
    for pool in s["pools"]:
        p = pool.view(torch.uint8) if pool.dtype in (torch.int8, torch.float8_e4m3fn) else pool
        unit = page // p.shape[2]  # rows per entry
        some = torch.arange(p.shape[2], device="cuda") * unit < rows[:, None]
        some = some[:, None, :, None] if p.dim() == 4 else some[:, None]
        p[to] = torch.where(some, p[of], p[to])
    return {"table": now.view(B * W, J).int(), "lens": lens.view(-1).int(), "pools": s["pools"]}


# ------------------------------------------------------------------ the work a pass cannot do without


def work(case):
    c = case
    if c["kind"] == "select":
        size = 4 if c["dtype"] == "fp32" else 2
        # Each logit is read, compared, and its exponential added up.
        return {"bytes": c["B"] * (c["W"] * (c["V"] * size + 4) + c["N"] * 16), "flops": 3 * c["B"] * c["W"] * c["V"]}
    if c["kind"] == "reorder":
        size = {"fp32": 4, "bf16": 2, "fp16": 2}.get(c["dtype"], 1)
        row = 2 * c["layers"] * c["Hkv"] * c["D"] * size
        # The rows of the pages in use of every second and later child of a beam; the tables, in and out.
        rows = sum(n % c["page"] * (c["W"] - len(set(p))) for n, p in zip(_lens(c), _parents(c)))
        return {"bytes": 2 * rows * row + 12 * c["B"] * c["W"] * -(-(c["L"] + 8) // c["page"]), "flops": 0}
    H, D = c["Hkv"], c["D"]
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "append":
        rows = sum(_counts(c))
        return {"bytes": 2 * H * (rows * D * (size + 1) + 4 * rows / RUN) + 4 * c["B"], "flops": 0}
    if c["kind"] == "read":
        rows = sum(max(0, min(n - f, c["N"])) for n, f in zip(_lens(c), _firsts(c)))
        return {"bytes": 2 * H * (rows * (D + 4 / RUN) + c["B"] * c["N"] * D * size), "flops": 0}
    new = c["B"] * c["T"] * D
    rows = sum(_lens(c))
    return {"bytes": 2 * rows * H * (D + 4 / RUN) + size * (2 * new * H + 2 * new * c["Hq"]),
            "flops": 4 * D * c["Hq"] * c["T"] * (rows + c["B"])}


# ------------------------------------------------------------------ the results in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "append": _exact_append, "read": _exact_read, "select": _exact_select,
            "reorder": _exact_reorder}[case["kind"]](s)


def _sequence(s, name, b, n):
    """(Hkv, n, D) in fp64: the first n rows of sequence b."""
    c = s["case"]
    codes, scales = s[name + "_codes"], s[name + "_scale"]
    units = [b] if c["page"] == 0 else s["table"][b].tolist()[:max(1, -(-n // c["page"]))]
    x = torch.cat([codes[u].double() * scales[u].double().repeat_interleave(RUN, 1)[:, :codes.shape[2], None] for u in units], 1)
    return x[:, :n]


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
        kc, vc = _sequence(s, "k", b, lens[b]), _sequence(s, "v", b, lens[b])
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


def _exact_code(x, fmt):
    """The nearest code of every value of x (fp64): ties to the even one."""
    if fmt == "int8":
        return torch.round(x)
    # e4m3: three bits behind the leading one, from 2^-6 on; below it steps of 2^-9.
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    c = s["case"]
    lens, counts = _lens(c), _counts(c)
    most = 448.0 if c["format"] == "e4m3" else 127.0
    out = {}
    for name in ("k", "v"):
        new = s[name].double().cpu()
        codes, scales = s[name + "_codes"][:-1].cpu().double(), s[name + "_scale"][:-1].cpu().double()
        for b in range(c["B"]):
            at = lens[b]
            while at < lens[b] + counts[b]:
                end = min(lens[b] + counts[b], at // RUN * RUN + RUN)
                src = [i - lens[b] if s["rows"] is None else int(s["rows"][b, i - lens[b]]) for i in range(at, end)]
                unit, row = (b, at) if c["page"] == 0 else (int(s["table"][b, at // c["page"]]), at % c["page"])
                j, first = row // RUN, row // RUN * RUN
                x = new[b][:, src]
                top = x.abs().amax((1, 2))
                was = scales[unit, :, j].clone() if row > first else torch.full_like(top, 2.0 ** LEAST)
                scale = torch.maximum(was, torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-9))) - 12))
                while (scale * most < top).any():
                    scale = torch.where(scale * most < top, 2 * scale, scale)
                codes[unit, :, first:row] = _exact_code(codes[unit, :, first:row] * (was / scale)[:, None, None], c["format"])
                codes[unit, :, row:row + end - at] = _exact_code(x / scale[:, None, None], c["format"])
                scales[unit, :, j] = scale
                at = end
        out[name + "_codes"] = codes.cuda() if c["format"] == "e4m3" else codes.to(torch.int8).cuda()
        out[name + "_scale"] = scales.cuda()
    return out


def _exact_read(s):
    c = s["case"]
    out = {}
    for name in ("k", "v"):
        x = torch.zeros((c["B"], c["Hkv"], c["N"], c["D"]), dtype=torch.float64, device="cuda")
        for b, (n, first) in enumerate(zip(_lens(c), _firsts(c))):
            n = max(0, min(n - first, c["N"]))
            x[b, :, :n] = _sequence(s, name, b, first + n)[:, first:]
        out[name] = x
    return out


def _exact_select(s):
    import numpy as np

    c = s["case"]
    scores, parents, tokens = [], [], []
    for b in range(c["B"]):
        found = []
        for w in range(c["W"]):
            base = float(s["scores"][b, w])
            if s["finished"] is not None and bool(s["finished"][b, w]):
                found.append((-base, w, 2))
                continue
            x = s["logits"][b, w].double().cpu().numpy()
            order = np.argsort(-x, kind="stable")[:c["N"]]
            top = x[order[0]]
            below = top + math.log(np.exp(x - top).sum())
            found += [(-(base + x[i] - below), w, int(i)) for i in order if x[i] > -math.inf]
        found = sorted(found)[:c["N"]]
        found += [(math.inf, 0, -1)] * (c["N"] - len(found))
        scores.append([-f[0] for f in found])
        parents.append([f[1] for f in found])
        tokens.append([f[2] for f in found])
    return {"scores": torch.tensor(scores, dtype=torch.float64, device="cuda"),
            "parents": torch.tensor(parents, dtype=torch.int32, device="cuda"), "tokens": torch.tensor(tokens, device="cuda")}


def _exact_reorder(s):
    """Whole numbers and copies, which have no other values in 64 bits: the pools after the moves that the tables say."""
    c = s["case"]
    B, W, page = c["B"], c["W"], c["page"]
    held, home, lens, par = (s[x].tolist() for x in ("table", "pages", "lens", "parents"))
    J = len(home[0])
    table = [[0] * J for _ in range(B * W)]
    moves = []
    for g in range(B):
        beams = range(g * W, g * W + W)
        n = [lens[g * W + par[g][i]] for i in range(W)]
        for j in range(J):
            fill = [max(0, min(page, x - j * page)) for x in n]
            want = [held[g * W + par[g][i]][j] for i in range(W)]
            whole = {want[i] for i in range(W) if fill[i] == page}
            kept = set(whole)
            stays = []
            for i in range(W):
                stay = fill[i] == page or (fill[i] > 0 and want[i] not in kept)
                stays.append(stay)
                if stay:
                    kept.add(want[i])
            free = [home[b][j] for b in beams if home[b][j] not in kept]
            for i in range(W):
                table[g * W + i][j] = want[i] if stays[i] else free.pop(0)
                if not stays[i] and fill[i]:
                    moves.append((want[i], table[g * W + i][j], fill[i]))
    pools = [p.clone() for p in s["pools"]]
    for p, new in zip(s["pools"], pools):
        for a, b, rows in moves:
            n = -(-rows * p.shape[2] // page)
            new[b][:, :n] = p[a][:, :n]
    new_lens = [lens[g * W + par[g][i]] for g in range(B) for i in range(W)]
    return {"table": torch.tensor(table, dtype=torch.int32, device="cuda"),
            "lens": torch.tensor(new_lens, dtype=torch.int32, device="cuda"), "pools": pools}
