"""Beam search and 8-bit caches run together, as a GPT serves with them.  Needs an MI355X.

The fp32 model is compared with its full forward on the CPU with the oracle attention.  Tolerance of a logit: each of the 9
products on a way through the two-layer model sums at most 512 terms, so fp32 moves it by at most 512 * 2^-24 = 2^-15 of its sum
of magnitudes; normalised activations are of size 1, the head sums 128 of them times weights of 0.016 on average (1.6 on average
before any sign): on both sides together 2 * 9 * 2^-15 * 2.1 < 1.2e-3.
"""
import copy
import math

import pytest
import torch

from co_alibi_attn import (co_alibi_attention, co_alibi_beam_select, co_alibi_cache_append_8bit, co_alibi_cache_read_8bit,
                           co_alibi_cache_reorder, co_alibi_decode_tree_8bit)
from co_alibi_attn import gpt as gpt_module
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref
from oracle import serving8 as oracle8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CFG = GPTConfig(n_layer=2, n_head=2, d_model=128, vocab=97)
TOL = 1.2e-3
FORMATS = (torch.float8_e4m3fn, torch.int8)


def oracle_attention(q, k, v, causal=True, sm_scale=None, bias_max=8.0):
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return ref.forward_autograd(q.float(), k.float(), v.float(), lam, causal=causal, scale=sm_scale).to(q.dtype)


@pytest.fixture(scope="module")
def models():
    torch.manual_seed(0)
    cpu = GPT(CFG, attention=oracle_attention)
    gpu = copy.deepcopy(cpu)
    for blk in gpu.blocks:
        blk.attn.attention = co_alibi_attention
    return cpu, gpu.to(DEV)


def logits_after(cpu):
    def run(tokens):
        with torch.no_grad():
            return cpu(torch.tensor([tokens]))[0, -1].double()
    return run


def prompts(lengths, seed, vocab=CFG.vocab):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (len(lengths), max(lengths)), generator=gen)


def recorded(monkeypatch):
    """The list that every selection's (scores, parents, tokens) from here on are put into, on the CPU."""
    steps, select = [], gpt_module.co_alibi_beam_select

    def record(*args):
        out = select(*args)
        steps.append(tuple(x.cpu() for x in out))
        return out

    monkeypatch.setattr(gpt_module, "co_alibi_beam_select", record)
    return steps


@pytest.mark.parametrize("page,beams,n", [(16, 4, 6), (64, 3, 6), (16, 1, 3)])
def test_the_search_is_the_one_by_whole_forwards(models, monkeypatch, page, beams, n):
    cpu, gpu = models
    lengths = [14, 1, 70]
    idx = prompts(lengths, 1)
    steps = recorded(monkeypatch)
    cache = PagedCache(CFG, 3 * beams, 96, torch.float32, DEV, page_size=page)
    tokens, scores = (x.cpu() for x in gpu.beam_search(idx.to(DEV), torch.tensor(lengths, device=DEV), n, beams, cache))
    for b, m in enumerate(lengths):
        oracle8.check_search(logits_after(cpu), b, idx[b, :m].tolist(), tokens[b], scores[b], steps, TOL)
    assert cache.seq_lens.tolist() == [m + n - 1 for m in lengths for _ in range(beams)]
    got = gpu.extend(tokens[:, :, -1].reshape(-1, 1).to(DEV), cache)[:, 0].cpu().double()
    for r in range(3 * beams):
        b, i = divmod(r, beams)
        want = logits_after(cpu)(idx[b, :lengths[b]].tolist() + tokens[b, i].tolist())
        assert (got[r] - want).abs().max() <= TOL


def test_finished_beams_and_ones_without_continuations(models, monkeypatch):
    cpu, gpu = models
    idx = prompts([4, 4], 2)
    end = torch.topk(logits_after(cpu)(idx[0].tolist()), 2).indices[1].item()
    steps = recorded(monkeypatch)
    tokens, scores = (x.cpu() for x in gpu.beam_search(idx.to(DEV), None, 4, 3, PagedCache(CFG, 6, 32, torch.float32, DEV), end))
    for b in range(2):
        oracle8.check_search(logits_after(cpu), b, idx[b].tolist(), tokens[b], scores[b], steps, TOL, end)
    small = GPTConfig(n_layer=1, n_head=2, d_model=128, vocab=5)
    torch.manual_seed(2)
    model = GPT(small).to(DEV)
    tokens, scores = model.beam_search(idx.to(DEV) % 5, None, 1, 7, PagedCache(small, 14, 16, torch.float32, DEV, page_size=16))
    assert (tokens[:, 5:] == -1).all() and (scores[:, 5:] == -math.inf).all()
    assert sorted(tokens[1, :5, 0].tolist()) == [0, 1, 2, 3, 4]


def filled(cfg, cache):
    """An fp32 cache that holds what an 8-bit one does."""
    plain = PagedCache(cfg, cache.seq_lens.shape[0], cache.capacity, torch.float32, DEV, page_size=cache.page_size)
    plain.seq_lens.copy_(cache.seq_lens)
    plain.bound = cache.bound
    page = cache.page_size
    for i, layer in enumerate(plain.layers):
        for pool, x in zip(layer, cache.read(i, torch.float32, rows=cache.capacity)):
            B, H, n, D = x.shape
            pool.view(B, n // page, H, page, D).copy_(x.view(B, H, n // page, page, D).transpose(1, 2))
    return plain


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", (16, 64))
def test_a_forward_over_8_bits_is_the_one_over_what_they_hold(models, fmt, page):
    _, gpu = models
    lengths = [70, 1, 16]
    idx = prompts(lengths, 3).to(DEV)
    cache = PagedCache(CFG, 3, 96, fmt, DEV, page_size=page)
    gpu.prefill(idx, cache, torch.tensor(lengths, device=DEV))
    tok = prompts([5, 5, 5], 4).to(DEV)
    parents = torch.tensor([-1, 0, 0, 1, 2], device=DEV).expand(3, 5)
    for _ in range(3):
        got = gpu.extend(tok, cache, parents)
        assert (got - gpu.extend(tok, filled(CFG, cache), parents)).abs().max() <= TOL
        gpu.extend(tok, cache, parents)
        cache.accept(torch.tensor([[0, 1, 3], [0, 2, 4], [0, 1, 1]], device=DEV), torch.tensor([3, 2, 0], device=DEV))
    assert cache.seq_lens.tolist() == [79, 7, 16]
    cache.clear()
    h = gpu.prefill(idx, cache, torch.tensor(lengths, device=DEV))
    assert torch.isfinite(h).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("autocast", (False, True))
def test_a_search_over_8_bits_is_the_one_that_copies_whole_caches(models, fmt, autocast, monkeypatch):
    cfg, gpu = CFG, models[1]
    if autocast:  # the benchmark model's shape
        cfg = GPTConfig(n_layer=2)
        torch.manual_seed(1)
        gpu = GPT(cfg).to(DEV)
    lengths = [15, 3, 40]
    idx, dev_len = prompts(lengths, 5, cfg.vocab).to(DEV), torch.tensor(lengths, device=DEV)

    def search():
        with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
            return gpu.beam_search(idx, dev_len, 8, 4, PagedCache(cfg, 12, 64, fmt, DEV, page_size=16))

    def by_copies(self, parents):
        heirs = (parents.long() + torch.arange(3, device=DEV)[:, None] * 4).view(-1)
        for t in (t for pair in self.layers + self.scales for t in pair):
            raw = t.view(torch.uint8) if t.dtype != torch.float32 else t
            raw.copy_(raw.view(12, 4, *t.shape[1:])[heirs].reshape(t.shape))
        self.seq_lens.copy_(self.seq_lens[heirs])

    got = search()
    monkeypatch.setattr(PagedCache, "reorder", by_copies)
    want = search()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isfinite(got[1]).all() and (got[0] >= 0).all()


@pytest.mark.parametrize("fmt", (torch.float32,) + FORMATS)
def test_a_captured_step_searches_token_after_token(models, fmt):
    _, gpu = models
    B, W, n = 2, 3, 10
    idx = prompts([12, 12], 6).to(DEV)
    want, want_scores = gpu.beam_search(idx, None, n, W, PagedCache(CFG, B * W, 64, fmt, DEV, page_size=16))
    cache = PagedCache(CFG, B * W, 64, fmt, DEV, page_size=16)
    logits = gpu.prefill(idx, cache.every(W))
    cache.bound = 12
    scores, parents, tok = co_alibi_beam_select(logits[:, None], torch.zeros(B, 1, device=DEV), W)
    cache.reorder(parents)

    def step():
        logits = gpu.extend(tok.view(B * W, 1), cache).view(B, W, -1)
        cache.accept()
        s, p, t = co_alibi_beam_select(logits, scores)
        cache.reorder(p)
        scores.copy_(s)
        parents.copy_(p)
        tok.copy_(t)

    state = [scores, parents, tok, cache.seq_lens, cache.block_table]
    saved = [x.clone() for x in state]
    pools = [t for pair in cache.layers + cache.scales for t in pair]
    kept = [t.clone() for t in pools]
    side = torch.cuda.Stream()  # warm-up off the capture, then back to the state before it
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(state + pools, saved + kept):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    steps = [(parents.cpu().long(), tok.cpu())]
    for _ in range(1, n):
        graph.replay()
        steps.append((parents.cpu().long(), tok.cpu()))
    out = torch.empty(B, W, n, dtype=torch.long)
    beam = torch.arange(W).expand(B, W)
    for i in reversed(range(n)):
        out[:, :, i] = steps[i][1].gather(1, beam)
        beam = steps[i][0].gather(1, beam)
    assert torch.equal(out, want.cpu()) and torch.equal(scores, want_scores)
    assert cache.seq_lens.tolist() == [12 + n - 1] * (B * W)


def step_inputs(fmt):
    gen = torch.Generator(device=DEV).manual_seed(20)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k, v = n(4, 4, 3, 64), n(4, 2, 3, 64), n(4, 2, 3, 64)
    caches = [(n(16, 2, 16, 64) * 20).to(fmt) for _ in range(2)]
    scales = [torch.full((16, 2, 1), 2.0 ** -4, device=DEV) for _ in range(2)]
    table = torch.arange(16, dtype=torch.int32, device=DEV).view(4, 4)
    lens = torch.tensor([40, 7, 0, 32], dtype=torch.int32, device=DEV)
    return q, k, v, *caches, *scales, table, lens


@pytest.mark.parametrize("fmt", FORMATS)
def test_operators_pass_the_dispatcher_checks(fmt):
    q, k, v, kc, vc, ks, vs, table, lens = step_inputs(fmt)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device=DEV)
    op = torch.ops.co_alibi
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV)
    # (The schema check compares inputs before and after, which torch has no e4m3 kernels for.)
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic") if fmt == torch.int8 else ("test_faketensor",)
    for args in ((q, k, v, kc, vc, ks, vs, slopes, lens, parents, table, 64, 0.125, True),
                 (q, k, v, kc, vc, ks, vs, slopes, None, None, table, 30, 0.125, False)):
        torch.library.opcheck(op.decode_tree_8bit.default, args, test_utils=checks)
    torch.library.opcheck(op.cache_append_8bit.default, (k, v, kc, vc, ks, vs, lens, None, None, table),
                          test_utils=checks)
    torch.library.opcheck(op.cache_read_8bit.default, (kc, vc, ks, vs, lens, None, table, 20, torch.float16),
                          test_utils=checks)
    logits = torch.randn(2, 2, 97, device=DEV)
    torch.library.opcheck(op.beam_select.default, (logits, torch.zeros(2, 2, device=DEV), None, 3, 0))
    torch.library.opcheck(op.cache_reorder.default, ([ks, vs], table, table.clone(), lens,
                                                     torch.tensor([[1, 1], [0, 0]], device=DEV), 16))


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_compiled_step_is_the_eager_one(fmt):
    head = torch.randn(64, 97, device=DEV)

    def step(q, k, v, kc, vc, ks, vs, table, lens):
        o = co_alibi_decode_tree_8bit(q, k, v, kc, vc, ks, vs, seq_len=lens, block_table=table)
        co_alibi_cache_append_8bit(k, v, kc, vc, ks, vs, lens, table)
        lens = lens + 3
        got = co_alibi_cache_read_8bit(kc, vc, ks, vs, lens, 43, torch.float32, table)
        scores, parents, tokens = co_alibi_beam_select((o.sum((1, 2)) @ head).view(2, 2, 97), torch.zeros(2, 2, device=DEV))
        new_table, new_lens = co_alibi_cache_reorder([kc, vc, ks, vs], lens, parents, table, table, 16)
        more = co_alibi_decode_tree_8bit(q, k, v, kc, vc, ks, vs, seq_len=new_lens, block_table=new_table)
        return o, more, *got, scores, parents, tokens, new_table, new_lens

    a, b = step_inputs(fmt), step_inputs(fmt)
    want = step(*a)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*b)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    for x, y in zip(a[3:7], b[3:7]):
        x, y = (t.view(torch.uint8) if t.dtype != torch.float32 else t for t in (x, y))
        assert torch.equal(x, y)
    assert torch.isfinite(want[1]).all()


@pytest.mark.parametrize("fmt", (torch.float32, torch.int8))
def test_inference_mode_and_an_empty_batch(models, fmt):
    _, gpu = models
    idx = prompts([18, 18], 8).to(DEV)
    want = gpu.beam_search(idx, None, 4, 3, PagedCache(CFG, 6, 32, fmt, DEV, page_size=16))
    with torch.inference_mode():
        got = gpu.beam_search(idx, None, 4, 3, PagedCache(CFG, 6, 32, fmt, DEV, page_size=16))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    tokens, scores = gpu.beam_search(idx[:0], None, 4, 3, PagedCache(CFG, 0, 32, fmt, DEV, page_size=16))
    assert tokens.shape == (0, 3, 4) and scores.shape == (0, 3)


@pytest.mark.parametrize("fmt", FORMATS)
def test_generation_and_drafts_over_8_bits(models, fmt):
    """A tree of one node is generate's step: the same cache, and so the same tokens."""
    _, gpu = models
    lengths = torch.tensor([20, 3], device=DEV)
    idx = prompts([20, 3], 9).to(DEV)
    u = torch.rand(2, 8, generator=torch.Generator().manual_seed(10)).to(DEV)
    cache = PagedCache(CFG, 2, 48, fmt, DEV, page_size=16)
    truth = gpu.generate(idx, lengths, u, cache)
    assert ((truth >= 0) & (truth < CFG.vocab)).all() and cache.seq_lens.tolist() == [27, 10]
    cache.clear()
    gpu.prefill(idx, cache, lengths)
    parents = torch.tensor([[-1], [-1]], device=DEV)
    for i in range(7):  # trees of one node: the draw of generate
        rows, counts, after = gpu.speculate(truth[:, i:i + 1], parents, u[:, i + 1:i + 2], cache)
        assert counts.tolist() == [1, 1] and torch.equal(after, truth[:, i + 1])
    wrong = (truth[:, :1] + 1) % CFG.vocab
    rows, counts, after = gpu.speculate(torch.cat([truth[:, 7:], wrong], 1), torch.tensor([[-1, 0], [-1, 0]], device=DEV),
                                        torch.zeros(2, 2, device=DEV), cache)
    assert ((counts == 1) | (after >= 0)).all() and cache.seq_lens.tolist() == [27 + counts[0], 10 + counts[1]]
