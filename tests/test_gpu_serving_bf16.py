"""The GPT's attention over a cache in bf16 under autocast: what each layer's call gave, from that call's own inputs, within
the oracle's bound; and the rows that it left in the cache, bit for bit.  Needs an MI355X."""
import pytest
import torch

from co_alibi_attn import gpt as gpt_module
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_each_layers_attention_under_autocast(monkeypatch):
    torch.manual_seed(1)
    cfg = GPTConfig(n_layer=2)
    gpu = GPT(cfg).to(DEV)
    with torch.no_grad():
        for blk in gpu.blocks:
            blk.attn.qkv.weight.mul_(4.0)  # scores of size 1, as a trained model has them
    idx = torch.randint(0, cfg.vocab, (2, 150), generator=torch.Generator().manual_seed(8)).to(DEV)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 1, 2, 3, 4, 5]], dtype=torch.int32)
    cache = PagedCache(cfg, 2, 192, torch.bfloat16, DEV)
    calls, native = [], gpt_module.co_alibi_decode_tree

    def recording(q, k, v, kc, vc, **kw):
        o = native(q, k, v, kc, vc, **kw)
        calls.append(([t.cpu() for t in (q, k, v, kc, vc)], kw["seq_len"].tolist(), o.cpu()))
        return o

    monkeypatch.setattr(gpt_module, "co_alibi_decode_tree", recording)
    lengths = [140, 61]
    with torch.autocast("cuda", torch.bfloat16):
        gpu.prefill(idx[:, :140], cache, torch.tensor(lengths, device=DEV))
        gpu.extend(idx[:, 143:], cache, parents.to(DEV))
    prefilled = [t.cpu() for layer in cache.layers for t in layer]
    new = [(k.cpu(), v.cpu()) for k, v in cache.new]
    cache.accept(torch.tensor([[0, 2, 5], [0, 1, 2]], device=DEV), torch.tensor([3, 1], device=DEV))
    lam = ref.slopes(cfg.n_head, cfg.bias_max, dtype=torch.bfloat16).float()
    half = torch.finfo(torch.bfloat16).eps / 2
    assert len(calls) == cfg.n_layer
    for (inputs, lens, o), (k, v) in zip(calls, new):
        assert lens == lengths and o.dtype == torch.bfloat16
        assert torch.equal(inputs[1], k) and torch.equal(inputs[2], v)
        want, _, bound, _ = oracle.decode_tree(*inputs, lens, parents, cache.block_table.cpu(), lam, 64 ** -0.5)
        assert ((o.double() - want).abs() - (half * (want.abs() + bound) + bound)).max() <= 0
    for i, (k, v) in enumerate(new):
        want = oracle.cache_append(k, v, *prefilled[2 * i:2 * i + 2], lengths, cache.block_table.cpu(),
                                   torch.tensor([[0, 2, 5], [0, 1, 2]]), [3, 1])
        for a, b in zip(want, cache.layers[i]):
            assert torch.equal(a, b.cpu())
