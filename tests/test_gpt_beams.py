"""GPT's beam search and its 8-bit caches on the CPU: the operators are replaced by the oracles, so what is tested is the
model's own bookkeeping -- forks, tables, finished beams, the way back through the parents."""
import math

import pytest
import torch

from co_alibi_attn import gpt as gpt_module
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref
from oracle import serving as oracle
from oracle import serving8 as oracle8

CFG = GPTConfig(n_layer=2, n_head=2, d_model=32, vocab=29)
FORMATS = (torch.float8_e4m3fn, torch.int8)
# Both sides run the same fp32 products, in another order: 9 of them on the way, sums of at most 128 terms, normalised
# activations of size 1 and a head whose 32 terms of 0.016 sum to 0.5 before any sign: 2 * 9 * 128 * 2^-24 * 0.5 < 7e-5.
TOL = 7e-5


def attention(q, k, v, causal=True, sm_scale=None, bias_max=8.0):
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return ref.forward_autograd(q.float(), k.float(), v.float(), lam, causal=causal, scale=sm_scale).to(q.dtype)


def attention_qkv(qkv, causal=True, bias_max=8.0):
    return attention(*(qkv[:, :, i].transpose(1, 2) for i in range(3)), causal=causal, bias_max=bias_max).transpose(1, 2)


def decode_tree(q, k, v, k_cache, v_cache, seq_len=None, parents=None, block_table=None, bias_max=8.0):
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return oracle.decode_tree(q, k, v, k_cache, v_cache, seq_len.tolist(), parents, block_table, lam,
                              q.shape[3] ** -0.5)[0].to(q.dtype)


def decode_tree_8bit(q, k, v, k_cache, v_cache, k_scale, v_scale, seq_len=None, parents=None, block_table=None, bias_max=8.0):
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return oracle8.decode_tree(q, k, v, (k_cache, v_cache), (k_scale, v_scale), seq_len.tolist(), parents, block_table, lam,
                               q.shape[3] ** -0.5)[0].to(q.dtype)


def cache_append(k, v, k_cache, v_cache, seq_lens, block_table=None, rows=None, counts=None):
    for old, new in zip((k_cache, v_cache), oracle.cache_append(k, v, k_cache, v_cache, seq_lens, block_table, rows, counts)):
        old.copy_(new)


def cache_append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, seq_lens, block_table=None, rows=None, counts=None):
    codes, scales = oracle8.append(k, v, (k_cache, v_cache), (k_scale, v_scale), seq_lens, block_table, rows, counts)
    for old, new in zip((k_cache, v_cache, k_scale, v_scale), codes + scales):
        old.copy_(new)


def cache_read_8bit(k_cache, v_cache, k_scale, v_scale, seq_lens, rows, dtype, block_table=None, first=None):
    return tuple(x.to(dtype) for x in oracle8.read((k_cache, v_cache), (k_scale, v_scale), seq_lens, block_table, first, rows))


def beam_select(logits, scores, num_beams=None, finished=None, end_token=0):
    s, p, t = oracle8.beam_select(logits, scores, num_beams or logits.shape[1], finished, end_token)
    return torch.tensor(s, dtype=torch.float64).float(), torch.tensor(p, dtype=torch.int32), torch.tensor(t)


def cache_reorder(caches, seq_lens, parents, block_table, pages, page_size=None):
    out, table, lens = oracle8.reorder([c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c for c in caches],
                                       block_table, pages, seq_lens, parents, page_size)
    for old, new in zip(caches, out):
        old.copy_(new.view(old.dtype))
    return table, lens


@pytest.fixture()
def model(monkeypatch):
    for name, f in (("attention_qkv", attention_qkv), ("decode_tree", decode_tree), ("decode_tree_8bit", decode_tree_8bit),
                    ("cache_append", cache_append), ("cache_append_8bit", cache_append_8bit),
                    ("cache_read_8bit", cache_read_8bit), ("beam_select", beam_select), ("cache_reorder", cache_reorder)):
        monkeypatch.setattr(gpt_module, "co_alibi_" + name, f)
    torch.manual_seed(0)
    return GPT(CFG, attention=attention)


def new_cache(batch, capacity=48, dtype=torch.float32):
    return PagedCache(CFG, batch, capacity, dtype, "cpu", page_size=16)


def prompts(lengths, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, CFG.vocab, (len(lengths), max(lengths)), generator=gen), torch.tensor(lengths)


def logits_after(model, tokens):
    with torch.no_grad():
        return model(torch.tensor([tokens]))[0, -1].double()


def recorded(monkeypatch):
    """The list that every selection's (scores, parents, tokens) from here on are put into."""
    steps, select = [], gpt_module.co_alibi_beam_select

    def record(*args):
        steps.append(select(*args))
        return steps[-1]

    monkeypatch.setattr(gpt_module, "co_alibi_beam_select", record)
    return steps


@pytest.mark.parametrize("beams,n,seed", [(1, 4, 1), (3, 5, 1), (4, 1, 1)])
def test_the_search_is_the_one_by_whole_forwards(model, monkeypatch, beams, n, seed):
    idx, lengths = prompts([14, 3], seed)
    steps = recorded(monkeypatch)
    cache = new_cache(2 * beams)
    tokens, scores = model.beam_search(idx, lengths, n, beams, cache)
    for b in range(2):
        oracle8.check_search(lambda seq: logits_after(model, seq), b, idx[b, :lengths[b]].tolist(), tokens[b], scores[b], steps, TOL)
    assert cache.seq_lens.tolist() == [x + n - 1 for x in lengths.tolist() for _ in range(beams)]
    # The cache's sequences are the beams: a forward behind each one's last token.
    got = model.extend(tokens[:, :, -1].reshape(-1, 1), cache)[:, 0].double()
    for r in range(2 * beams):
        b, i = divmod(r, beams)
        want = logits_after(model, idx[b, :lengths[b]].tolist() + tokens[b, i].tolist())
        assert (got[r] - want).abs().max() <= TOL


def test_finished_beams_keep_their_scores(model, monkeypatch):
    idx, lengths = prompts([4], 2)
    first = torch.log_softmax(logits_after(model, idx[0].tolist()), 0).topk(3).indices
    end = first[1].item()  # the second beam ends at once
    steps = recorded(monkeypatch)
    tokens, scores = model.beam_search(idx, lengths, 4, 3, new_cache(3), end_token=end)
    oracle8.check_search(lambda seq: logits_after(model, seq), 0, idx[0].tolist(), tokens[0], scores[0], steps, TOL, end)
    assert [end] * 4 in tokens[0].tolist()


def test_more_beams_than_continuations(model):
    idx, lengths = prompts([2, 2], 3)
    tokens, scores = model.beam_search(idx, None, 1, 40, new_cache(80, 16))
    assert (tokens[:, 29:] == -1).all() and (scores[:, 29:] == -math.inf).all()
    for b in range(2):
        assert sorted(tokens[b, :29, 0].tolist()) == list(range(29))
        assert scores[b, :29].double().exp().sum().item() == pytest.approx(1, abs=29 * 2.0 ** -24 * 4)
    tokens, scores = model.beam_search(idx, None, 2, 40, new_cache(80, 16))  # the next step has enough
    assert (tokens >= 0).all() and torch.isfinite(scores).all()


def test_a_prompt_without_continuations(model):
    """Logits of NaN: the beams are dead from the start, and the other prompt's are not."""
    with torch.no_grad():
        model.wte.weight[7] = math.nan
    idx, lengths = prompts([5, 5], 4)
    idx[idx == 7] = 8
    idx[0, 2] = 7
    with pytest.MonkeyPatch.context() as m:  # a head without that row
        sane = model.wte.weight.detach().clone()
        sane[7] = 0
        linear = gpt_module.F.linear
        m.setattr(gpt_module.F, "linear", lambda x, w, b=None: linear(x, sane if w is model.wte.weight else w, b))
        tokens, scores = model.beam_search(idx, None, 3, 2, new_cache(4))
    assert (tokens[0] == -1).all() and (scores[0] == -math.inf).all()
    assert (tokens[1] >= 0).all() and torch.isfinite(scores[1]).all()


def test_a_cleared_cache_serves_again(model):
    idx, lengths = prompts([17, 3])  # (17 rows: the beams share a full page)
    cache = new_cache(6)
    want = model.beam_search(idx, lengths, 5, 3, cache)
    with pytest.raises(ValueError, match="empty cache"):
        model.beam_search(idx, lengths, 5, 3, cache)
    assert not torch.equal(cache.block_table, cache.pages)
    cache.clear()
    assert torch.equal(cache.block_table, cache.pages) and cache.seq_lens.tolist() == [0] * 6
    got = model.beam_search(idx, lengths, 5, 3, cache)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(model):
    idx, lengths = prompts([4, 3])
    for n, beams, batch, end, match in ((0, 3, 6, None, "at least one token"), (2, 3, 5, None, "cache of as many"),
                                        (2, 0, 0, None, "1 to 64"), (2, 65, 130, None, "1 to 64"),
                                        (2, 3, 6, 29, "end_token"), (2, 3, 6, -1, "end_token")):
        with pytest.raises(ValueError, match=match):
            model.beam_search(idx, lengths, n, beams, new_cache(batch, 16), end_token=end)
    with pytest.raises(ValueError, match="1 more rows behind 16 do not fit"):
        model.beam_search(idx, lengths, 14, 3, new_cache(6, 16))
    cache = new_cache(6)
    for bad in (torch.zeros(2, 2), torch.zeros(6)):
        with pytest.raises(ValueError, match="parents must be"):
            cache.reorder(bad.int())
    with pytest.raises(ValueError, match="8-bit caches"):
        cache.read(0)


def filled(cache, fmt):
    """An fp32 cache that holds what an 8-bit one does."""
    plain = PagedCache(CFG, cache.seq_lens.shape[0], cache.capacity, torch.float32, "cpu", page_size=16)
    plain.seq_lens.copy_(cache.seq_lens)
    plain.bound = cache.bound
    for i, layer in enumerate(plain.layers):
        for pool, x in zip(layer, cache.read(i, torch.float32)):
            for b in range(x.shape[0]):
                for r in range(cache.seq_lens[b]):
                    pool[plain.block_table[b, r // 16], :, r % 16] = x[b, :, r]
    return plain


@pytest.mark.parametrize("fmt", FORMATS)
def test_8_bit_caches(model, fmt):
    """What a forward over 8 bits gives is what one over the values read back gives."""
    idx, lengths = prompts([20, 1, 16], 5)
    cache = new_cache(3, dtype=fmt)
    model.prefill(idx, cache, lengths)
    assert all(c.dtype == fmt for layer in cache.layers for c in layer) and len(cache.scales) == 2
    tok = torch.tensor([[3, 4], [5, 6], [7, 8]])
    parents = torch.tensor([-1, 0]).expand(3, 2)
    got = model.extend(tok, cache, parents)
    assert (got - model.extend(tok, filled(cache, fmt), parents)).abs().max() <= TOL
    cache.accept(torch.tensor([[0, 1], [1, 0], [0, 0]]), torch.tensor([2, 1, 0]))
    assert cache.seq_lens.tolist() == [22, 2, 16]
    got = model.extend(tok, cache)
    assert (got - model.extend(tok, filled(cache, fmt))).abs().max() <= TOL
    k, v = cache.read(1, torch.float32, rows=3, first=torch.tensor([19, 0, 15]))
    want = cache.read(1, torch.float32)
    assert k.shape == (3, 2, 3, 16) and torch.equal(k[0], want[0][0, :, 19:22]) and torch.equal(v[1, :, :2], want[1][1, :, :2])
    assert (k[1, :, 2:] == 0).all() and (v[2, :, 1:] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_search_over_8_bits_is_the_one_that_copies_whole_caches(model, fmt, monkeypatch):
    idx, lengths = prompts([15, 3], 6)
    got = model.beam_search(idx, lengths, 4, 3, new_cache(6, dtype=fmt))

    def by_copies(self, parents):
        heirs = (parents.long() + torch.arange(2)[:, None] * 3).view(-1)
        for t in (t for pair in self.layers + self.scales for t in pair):
            t.copy_(t.view(6, 3, *t.shape[1:])[heirs].reshape(t.shape))
        self.seq_lens.copy_(self.seq_lens[heirs])

    monkeypatch.setattr(PagedCache, "reorder", by_copies)
    want = model.beam_search(idx, lengths, 4, 3, new_cache(6, dtype=fmt))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
