"""Cache, tree attention and sampling run together, as a GPT serves with them.  Needs an MI355X.

The fp32 model's logits over a cache are compared with its full forward on the CPU with the oracle attention.
Tolerance: each of the 9 products on a way through the two-layer model sums at most 512 terms, so fp32 moves it by at
most 512 * 2^-24 = 2^-15 of its sum of magnitudes; normalised activations are of size 1, the head sums 128 of them
times weights of 0.016 on average (1.6 on average before any sign): on both sides together 2 * 9 * 2^-15 * 2.1 < 1.2e-3.
A weight that a logit may move by that is moved by 1.2e-3 of itself, a border between two tokens by as much.
"""
import copy

import pytest
import torch

from co_alibi_attn import co_alibi_attention, co_alibi_cache_append, co_alibi_decode_tree, co_alibi_sample
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CFG = GPTConfig(n_layer=2, n_head=2, d_model=128, vocab=97)
TOL = 1.2e-3


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


def logits_after(cpu, tokens):
    """Logits behind the last of these tokens, by the full forward."""
    with torch.no_grad():
        return cpu(torch.tensor([tokens]))[0, -1].double()


def check_draw(logits, uniform, token):
    order = sorted(range(len(logits)), key=lambda i: (-logits[i].item(), i))
    p = torch.softmax(logits, 0)
    # Tokens whose logits the tolerance cannot tell apart may change places.
    before = sum(p[i].item() for i in order if logits[i] > logits[token] + 2 * TOL)
    upto = sum(p[i].item() for i in order if logits[i] >= logits[token] - 2 * TOL)
    assert before - TOL <= uniform <= upto + TOL, (before, uniform, upto, token)


def prompts(lengths, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, CFG.vocab, (len(lengths), max(lengths)), generator=gen)


@pytest.mark.parametrize("page", (16, 64))
def test_generate_follows_the_full_forward(models, page):
    cpu, gpu = models
    lengths = [1, 70, 16, 33]
    idx = prompts(lengths, 1)
    u = torch.rand(4, 20, generator=torch.Generator().manual_seed(2))
    cache = PagedCache(CFG, 4, 96, torch.float32, DEV, page_size=page)
    out = gpu.generate(idx.to(DEV), torch.tensor(lengths, device=DEV), u.to(DEV), cache).cpu()
    assert cache.seq_lens.tolist() == [n + 19 for n in lengths]
    for b, n in enumerate(lengths):
        seq = idx[b, :n].tolist()
        for i in range(20):
            check_draw(logits_after(cpu, seq), u[b, i].item(), out[b, i].item())
            seq.append(out[b, i].item())
    again = PagedCache(CFG, 4, 96, torch.float32, DEV, page_size=page)
    with torch.inference_mode():
        assert torch.equal(gpu.generate(idx.to(DEV), torch.tensor(lengths, device=DEV), u.to(DEV), again).cpu(), out)


def test_generate_at_temperature_0(models):
    cpu, gpu = models
    idx = prompts([5, 5], 3)
    cache = PagedCache(CFG, 2, 64, torch.float32, DEV)
    out = gpu.generate(idx.to(DEV), None, torch.zeros(2, 12, device=DEV), cache, temperature=0.0).cpu()
    for b in range(2):
        seq = idx[b].tolist()
        for i in range(12):
            want = logits_after(cpu, seq)
            assert want[out[b, i]] >= want.max() - 2 * TOL
            seq.append(out[b, i].item())


def test_tree_then_its_accepted_path(models):
    """Logits behind every node; the cache after a path is accepted, or the first rows, or all."""
    cpu, gpu = models
    lengths = [17, 40, 3]
    idx = prompts(lengths, 4)
    cache = PagedCache(CFG, 3, 128, torch.float32, DEV, page_size=16)
    first = gpu.prefill(idx.to(DEV), cache, torch.tensor(lengths, device=DEV)).cpu().double()
    seqs = [idx[b, :n].tolist() for b, n in enumerate(lengths)]
    for b in range(3):
        assert (first[b] - logits_after(cpu, seqs[b])).abs().max() <= TOL
    par = torch.tensor([[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 2, 3, 4, 5], [-1, -1, 0, 1, 3, 4, 4]], dtype=torch.int32)
    gen = torch.Generator().manual_seed(5)
    for step, (rows, counts) in enumerate([([[0, 2, 5, 6], [0, 1, 2, 0], [1, 3, 4, 6]], [4, 3, 4]),
                                           (None, [7, 0, 0]), ([[0, 1, 4, 4], [0, 1, 2, 3], [0, 2, 0, 0]], [3, 4, 2])]):
        tok = torch.randint(0, CFG.vocab, (3, 7), generator=gen)
        chain = step == 1
        got = gpu.extend(tok.to(DEV), cache, None if chain else par.to(DEV)).cpu().double()
        for b in range(3):
            for t in range(7):
                path, n = [], t
                while n >= 0:
                    path.insert(0, tok[b, n].item())
                    n = n - 1 if chain else int(par[b, n])
                assert (got[b, t] - logits_after(cpu, seqs[b] + path)).abs().max() <= TOL, (step, b, t)
            kept = range(counts[b]) if rows is None else rows[b][:counts[b]]
            seqs[b] += [tok[b, r].item() for r in kept]
        cache.accept(None if rows is None else torch.tensor(rows, device=DEV), torch.tensor(counts, device=DEV))
        assert cache.seq_lens.tolist() == [len(s) for s in seqs]
    tok = torch.randint(0, CFG.vocab, (3, 1), generator=gen)
    got = gpu.extend(tok.to(DEV), cache).cpu().double()
    for b in range(3):
        assert (got[b, 0] - logits_after(cpu, seqs[b] + tok[b].tolist())).abs().max() <= TOL


def test_speculation_gives_what_token_by_token_gives(models):
    cpu, gpu = models
    lengths = [9, 30, 1]
    idx = prompts(lengths, 6)
    dev_len = torch.tensor(lengths, device=DEV)
    u = torch.rand(3, 6, generator=torch.Generator().manual_seed(7))
    plain = PagedCache(CFG, 3, 64, torch.float32, DEV)
    truth = gpu.generate(idx.to(DEV), dev_len, u.to(DEV), plain).cpu()  # (3, 6)
    cache = PagedCache(CFG, 3, 64, torch.float32, DEV)
    gpu.prefill(idx.to(DEV), cache, dev_len)
    # Node 0 is truth[:, 0]; a wrong and a right child at each depth, the right one twice at depth 1.
    par = torch.tensor([-1, 0, 0, 0, 2, 2, 5, 5, 3]).expand(3, 9).contiguous()
    depth = torch.tensor([0, 1, 1, 1, 2, 2, 3, 3, 2])
    right = torch.tensor([1, 0, 1, 1, 0, 1, 1, 0, 1], dtype=torch.bool)
    tok = torch.where(right, truth[:, depth], (truth[:, depth] + 1) % CFG.vocab)
    tok[1, 5] = (tok[1, 5] + 2) % CFG.vocab  # sequence 1: its second draft is wrong
    tok[2, 2:4] = (tok[2, 2:4] + 3) % CFG.vocab  # sequence 2: all are wrong
    par[2, 8] = 9  # an absent node
    rows, counts, after = gpu.speculate(tok.to(DEV), par.to(DEV), u[:, 1:][:, depth].to(DEV), cache)
    assert counts.tolist() == [4, 2, 1]
    want = [[0, 2, 5, 6], [0, 2], [0]]
    for b in range(3):
        n = counts[b].item()
        assert rows[b, :n].tolist() == want[b]
        assert after[b].item() == truth[b, n].item()
        seq = idx[b, :lengths[b]].tolist() + truth[b, :n].tolist()
        check_draw(logits_after(cpu, seq), u[b, n].item(), after[b].item())
    assert cache.seq_lens.tolist() == [lengths[b] + counts[b].item() for b in range(3)]
    got = gpu.extend(after[:, None], cache).cpu().double()
    for b in range(3):
        seq = idx[b, :lengths[b]].tolist() + truth[b, :counts[b]].tolist() + [after[b].item()]
        assert (got[b, 0] - logits_after(cpu, seq)).abs().max() <= TOL


def test_bf16_autocast_serves(models):
    """The benchmark model's shape under autocast: extend over a cache against the full forward, both on the GPU."""
    torch.manual_seed(1)
    cfg = GPTConfig(n_layer=2)
    gpu = GPT(cfg).to(DEV)
    idx = torch.randint(0, cfg.vocab, (2, 300), generator=torch.Generator().manual_seed(8)).to(DEV)
    cache = PagedCache(cfg, 2, 320, torch.bfloat16, DEV)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        full = gpu(idx).float()
        a = gpu.prefill(idx[:, :280], cache)
        b = gpu.extend(idx[:, 280:], cache)
    # bf16 products: 17 of them on the way, each rounded by up to 2^-8 of itself, 0.55 being the logits' spread.
    assert (a.float() - full[:, 279]).abs().max() <= 17 * 2.0 ** -8 * 4 * 0.55
    assert (b.float() - full[:, 280:]).abs().max() <= 17 * 2.0 ** -8 * 4 * 0.55
    assert b.dtype == torch.bfloat16


def test_a_captured_step_serves_token_after_token(models):
    _, gpu = models
    idx = prompts([20, 20], 9).to(DEV)
    u = torch.rand(2, 9, generator=torch.Generator().manual_seed(10)).to(DEV)
    want = gpu.generate(idx, None, u, PagedCache(CFG, 2, 64, torch.float32, DEV))
    cache = PagedCache(CFG, 2, 64, torch.float32, DEV)
    tok = co_alibi_sample(gpu.prefill(idx, cache), u[:, 0])[:, None]
    uniform = torch.empty(2, device=DEV)

    def step():
        logits = gpu.extend(tok, cache)[:, 0]
        cache.accept()
        tok.copy_(co_alibi_sample(logits, uniform)[:, None])

    side = torch.cuda.Stream()  # warm-up off the capture, then back to the state before it
    side.wait_stream(torch.cuda.current_stream())
    saved, lens = tok.clone(), cache.seq_lens.clone()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    tok.copy_(saved)
    cache.seq_lens.copy_(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    got = [tok.clone()]
    for i in range(1, 9):
        uniform.copy_(u[:, i])
        graph.replay()
        got.append(tok.clone())
        torch.cuda.synchronize()
    assert torch.equal(torch.cat(got, 1), want)
    assert cache.seq_lens.tolist() == [28, 28]


def test_a_full_cache_is_refused(models):
    _, gpu = models
    cache = PagedCache(CFG, 1, 16, torch.float32, DEV, page_size=16)
    idx = prompts([16], 11).to(DEV)
    with pytest.raises(ValueError, match="do not fit"):
        gpu.prefill(torch.cat([idx, idx], 1), cache)
    gpu.prefill(idx[:, :14], cache, torch.tensor([10], device=DEV))
    with pytest.raises(ValueError, match="empty cache"):
        gpu.prefill(idx, cache)
    with pytest.raises(ValueError, match="at most 64 new tokens"):
        gpu.extend(idx[:, :1].expand(1, 65), cache)
    with pytest.raises(ValueError, match="no new keys"):  # of a forward that was refused
        cache.accept()
    gpu.extend(idx[:, :4], cache)  # 10 rows are filled, 14 were bounded
    cache.accept()
    gpu.extend(idx[:, :3], cache)
    before = [t.clone() for layer in cache.layers for t in layer]
    with pytest.raises(ValueError, match="3 more rows behind 14"):
        cache.accept()
    assert all(torch.equal(a, b) for a, b in zip(before, [t for layer in cache.layers for t in layer]))
    cache.accept(counts=torch.tensor([2], device=DEV))
    assert cache.seq_lens.tolist() == [16]
    o = co_alibi_decode_tree(*(torch.zeros(1, 2, 1, 64, device=DEV) for _ in range(3)), *cache.layers[0],
                             seq_len=cache.seq_lens, block_table=cache.block_table)
    assert torch.isfinite(o).all()


def step_inputs():
    gen = torch.Generator(device=DEV).manual_seed(20)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k, v = n(2, 4, 3, 64), n(2, 2, 3, 64), n(2, 2, 3, 64)
    pools = n(9, 2, 16, 64), n(9, 2, 16, 64)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    lens = torch.tensor([40, 7], dtype=torch.int32, device=DEV)
    return q, k, v, *pools, table, lens


def test_operators_pass_the_dispatcher_checks():
    q, k, v, kc, vc, table, lens = step_inputs()
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device=DEV)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV)
    op = torch.ops.co_alibi
    for args in ((q, k, v, kc, vc, slopes, lens, parents, table, 64, 0.125, True), (q, k, v, kc, vc, slopes, None, None, table, 30, 0.125, False)):
        torch.library.opcheck(op.decode_tree.default, args)
    counts = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    for args in ((k, v, kc, vc, lens, None, None, table), (k, v, kc, vc, lens, counts, torch.tensor([[0, 2], [1, 0]], device=DEV), table)):
        torch.library.opcheck(op.cache_append.default, args)
    logits, u = torch.randn(3, 500, device=DEV), torch.rand(3, device=DEV)
    torch.library.opcheck(op.sample.default, (logits, u, None, None, None, None, 0.9, 20, 0.95, 0.0))
    torch.library.opcheck(op.sample.default, (logits, u, u, None, u, None, 1.0, 0, 1.0, 0.1))


def test_a_compiled_step_is_the_eager_one():
    head = torch.randn(64, 97, device=DEV)

    def step(q, k, v, kc, vc, table, lens, u):
        o = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, block_table=table)
        co_alibi_cache_append(k, v, kc, vc, lens, table)
        more = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens + 3, block_table=table)
        return o, more, co_alibi_sample((o + more).sum((1, 2)) @ head, u, top_p=0.9)

    u = torch.rand(2, device=DEV)
    a, b = step_inputs(), step_inputs()
    want = step(*a, u)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*b, u)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    assert torch.equal(a[3], b[3]) and torch.equal(a[4], b[4])
    assert not torch.equal(a[3], step_inputs()[3])
