"""A captured serving step replayed until its cache is full, and beyond.  Needs an MI355X."""
import pytest
import torch

from co_alibi_attn import co_alibi_sample
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CFG = GPTConfig(n_layer=2, n_head=2, d_model=128, vocab=97)


def test_replays_fill_the_cache_and_eager_calls_see_it():
    torch.manual_seed(0)
    gpu = GPT(CFG).to(DEV)
    gen = torch.Generator().manual_seed(1)
    idx = torch.randint(0, CFG.vocab, (2, 20), generator=gen).to(DEV)
    u = torch.rand(2, 13, generator=gen).to(DEV)
    want = gpu.generate(idx, None, u, PagedCache(CFG, 2, 32, torch.float32, DEV, page_size=16))
    cache = PagedCache(CFG, 2, 32, torch.float32, DEV, page_size=16)
    tok = co_alibi_sample(gpu.prefill(idx, cache), u[:, 0])[:, None]
    uniform = torch.empty(2, device=DEV)

    def step():
        logits = gpu.extend(tok, cache)[:, 0]
        cache.accept()
        tok.copy_(co_alibi_sample(logits, uniform)[:, None])

    saved, side = tok.clone(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    tok.copy_(saved)
    cache.seq_lens.fill_(20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    got = [tok.clone()]
    for i in range(1, 13):  # the 12 rows that are left
        uniform.copy_(u[:, i])
        cache.room_for(1)
        graph.replay()
        got.append(tok.clone())
        torch.cuda.synchronize()
    assert torch.equal(torch.cat(got, 1), want) and cache.seq_lens.tolist() == [32, 32]
    with pytest.raises(ValueError, match="1 more rows behind 32"):
        cache.room_for(1)
    rows = [t.clone() for layer in cache.layers for t in layer]
    for _ in range(3):  # without looking
        graph.replay()
        torch.cuda.synchronize()
    assert cache.seq_lens.tolist() == [32, 32]
    assert all(torch.equal(a, b) for a, b in zip(rows, [t for layer in cache.layers for t in layer]))
    gpu.extend(tok, cache)
    with pytest.raises(ValueError, match="1 more rows behind 32"):
        cache.accept()
    with pytest.raises(ValueError, match="do not fit"):
        gpu.speculate(tok, torch.full((2, 1), -1, device=DEV), torch.zeros(2, 1, device=DEV), cache)
    with pytest.raises(ValueError, match="empty cache"):
        gpu.prefill(idx, cache)
