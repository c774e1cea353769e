"""GPT's serving path on the CPU: the four operators it calls are replaced by the oracles, so what is tested is the
model's own bookkeeping -- trees, rooms, lengths, and tokens that a draw could not give."""
import pytest
import torch

from co_alibi_attn import gpt as gpt_module
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref
from oracle import serving as oracle

CFG = GPTConfig(n_layer=2, n_head=2, d_model=32, vocab=29)


def attention(q, k, v, causal=True, sm_scale=None, bias_max=8.0):
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return ref.forward_autograd(q.float(), k.float(), v.float(), lam, causal=causal, scale=sm_scale).to(q.dtype)


def attention_qkv(qkv, causal=True, bias_max=8.0):
    return attention(*(qkv[:, :, i].transpose(1, 2) for i in range(3)), causal=causal, bias_max=bias_max).transpose(1, 2)


def decode_tree(q, k, v, k_cache, v_cache, seq_len=None, parents=None, block_table=None, bias_max=8.0):
    page, blocks = k_cache.shape[2], block_table.shape[1]
    lens = seq_len.clamp(0, page * blocks).tolist()
    lam = ref.slopes(q.shape[1], bias_max, dtype=q.dtype).float()
    return oracle.decode_tree(q, k, v, k_cache, v_cache, lens, parents, block_table, lam, q.shape[3] ** -0.5)[0].to(q.dtype)


def cache_append(k, v, k_cache, v_cache, seq_lens, block_table=None, rows=None, counts=None):
    for old, new in zip((k_cache, v_cache), oracle.cache_append(k, v, k_cache, v_cache, seq_lens, block_table, rows, counts)):
        old.copy_(new)


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    B = logits.shape[0]
    return torch.tensor(oracle.sample(logits, uniforms, [temperature] * B, [top_k] * B, [top_p] * B, [min_p] * B))


@pytest.fixture()
def model(monkeypatch):
    for name, f in (("co_alibi_attention_qkv", attention_qkv), ("co_alibi_decode_tree", decode_tree),
                    ("co_alibi_cache_append", cache_append), ("co_alibi_sample", sample)):
        monkeypatch.setattr(gpt_module, name, f)
    torch.manual_seed(0)
    return GPT(CFG, attention=attention)


def new_cache(batch, capacity=32):
    return PagedCache(CFG, batch, capacity, torch.float32, "cpu", page_size=16)


def start(model, lengths, drawn, capacity=32, seed=1):
    """Prompts, `drawn` uniform numbers behind each, and the tokens that drawing one by one gives with them."""
    gen = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, CFG.vocab, (len(lengths), max(lengths)), generator=gen)
    u = torch.rand(len(lengths), drawn, generator=gen)
    return idx, torch.tensor(lengths), u, model.generate(idx, torch.tensor(lengths), u, new_cache(len(lengths), 64))


def test_generate_follows_the_full_forward(model):
    """(That the replacements stand in for the operators.)"""
    idx, lengths, u, out = start(model, [5, 1], 6)
    for b in range(2):
        seq = idx[b, :lengths[b]].tolist()
        for i in range(6):
            with torch.no_grad():
                logits = model(torch.tensor([seq]))[:, -1]
            assert sample(logits, u[b:b + 1, i]).tolist() == [out[b, i].item()]
            seq.append(out[b, i].item())


def test_an_absent_node_is_no_earlier_twin(model):
    """Node 1's parent comes after it, so node 1 is absent; node 3 holds the same token behind the same, valid parent."""
    idx, lengths, u, truth = start(model, [4], 4)
    parents = torch.tensor([[-1, 2, 0, 2]])
    depth = torch.tensor([0, 2, 1, 2])
    cache = new_cache(1)
    model.prefill(idx, cache, lengths)
    rows, counts, after = model.speculate(truth[:, depth], parents, u[:, 1:][:, depth], cache)
    assert counts.tolist() == [3] and rows[0, :3].tolist() == [0, 2, 3] and after.tolist() == truth[:, 3].tolist()


def test_the_last_rows_of_a_cache_take_the_path_that_fits(model):
    """Room for fewer rows than the tree has nodes: what fits of the accepted path is kept, the next token is drawn behind it."""
    idx, lengths, u, truth = start(model, [29, 30, 31], 6)
    parents = torch.tensor([-1, 0, 0, 2, 3, 4]).expand(3, 6).contiguous()
    depth = torch.tensor([0, 1, 1, 2, 3, 4])
    tok = truth[:, depth].clone()
    tok[:, 1] = (tok[:, 1] + 1) % CFG.vocab
    cache = new_cache(3)
    model.prefill(idx, cache, lengths)
    rows, counts, after = model.speculate(tok, parents, u[:, 1:][:, depth], cache)
    path = [0, 2, 3, 4, 5]
    assert counts.tolist() == [3, 2, 1] and cache.seq_lens.tolist() == [32, 32, 32]
    for b, n in enumerate((3, 2, 1)):
        assert rows[b, :n].tolist() == path[:n] and after[b] == truth[b, n]
    with pytest.raises(ValueError, match="do not fit"):
        model.speculate(tok, parents, u[:, 1:][:, depth], cache)


def test_a_row_without_a_token_stays_without_one(model, monkeypatch):
    """-1 (a row of NaN, say) is no row of the embedding; what such a sequence would go on with is -1, too."""
    idx, lengths, u, truth = start(model, [3, 4], 5)
    calls = []

    def failing(logits, uniforms, **kw):
        out = sample(logits, uniforms, **kw)
        calls.append(0)
        if len(calls) == 2:
            out[1] = -1
        return out

    monkeypatch.setattr(gpt_module, "co_alibi_sample", failing)
    out = model.generate(idx, lengths, u, new_cache(2))
    assert out[0].tolist() == truth[0].tolist()
    assert out[1].tolist() == truth[1, :1].tolist() + [-1] * 4


def test_tokens_below_0_are_read_as_0(model):
    """What a caller feeds back after such a draw stays inside the embedding."""
    cache = new_cache(2)
    idx = torch.tensor([[3, 4], [5, 6]])
    assert torch.equal(model.prefill(torch.tensor([[3, 4], [-1, 6]]), cache)[0], model.prefill(idx, new_cache(2))[0])
    got = model.extend(torch.tensor([[7], [-1]]), cache)
    want = model.extend(torch.tensor([[7], [0]]), cache)
    assert torch.equal(got, want) and torch.isfinite(got).all()


def test_prompt_lengths_outside_the_prompts_are_clamped(model):
    idx = torch.randint(0, CFG.vocab, (3, 6), generator=torch.Generator().manual_seed(3))
    cache, want_cache = new_cache(3), new_cache(3)
    got = model.prefill(idx, cache, torch.tensor([0, 9, 1 << 40]))
    want = model.prefill(idx, want_cache, torch.tensor([1, 6, 6]))
    assert torch.equal(got, want) and cache.seq_lens.tolist() == want_cache.seq_lens.tolist() == [1, 6, 6]
    with pytest.raises(ValueError, match="at least one token"):
        model.prefill(idx[:, :0], new_cache(3), torch.tensor([1, 1, 1]))


def test_replays_of_a_captured_step_are_counted(model, monkeypatch):
    """A replayed accept moves the lengths without the host: from the capture on the room is read from the device, and a
    replay that finds none leaves the lengths at the capacity."""
    cache = new_cache(2)
    model.prefill(torch.tensor([[1, 2, 3], [4, 5, 6]]), cache)
    tok = torch.tensor([[7], [8]])

    def step():
        model.extend(tok, cache)
        cache.accept()

    monkeypatch.setattr(PagedCache, "_capturing", lambda self: True, raising=False)
    step()  # stands for the capture, which runs the host's part once ...
    for _ in range(28):  # ... and for the replays, of which the host sees nothing
        bound = cache.bound
        step()
        cache.bound = bound
    assert cache.seq_lens.tolist() == [32, 32]
    step()
    assert cache.seq_lens.tolist() == [32, 32]
    monkeypatch.undo()
    for name, f in (("co_alibi_decode_tree", decode_tree), ("co_alibi_cache_append", cache_append)):
        monkeypatch.setattr(gpt_module, name, f)
    with pytest.raises(ValueError, match="1 more rows behind 32 do not fit"):
        step()
    with pytest.raises(ValueError, match="empty cache"):
        model.prefill(torch.tensor([[1], [2]]), cache)
    cache.seq_lens.zero_()
    cache.room_for(32)
    assert cache.bound == 0


def test_no_draft_is_accepted_where_no_token_was_drawn(model, monkeypatch):
    """A draft of -1 behind a node whose draw gave -1 is no token that was drawn."""
    idx, lengths, u, truth = start(model, [3], 2)
    monkeypatch.setattr(gpt_module, "co_alibi_sample", lambda logits, uniforms, **kw: torch.full((logits.shape[0],), -1))
    cache = new_cache(1)
    model.prefill(idx, cache, lengths)
    rows, counts, after = model.speculate(torch.tensor([[truth[0, 0], -1]]), torch.tensor([[-1, 0]]), u, cache)
    assert counts.tolist() == [1] and rows[0, 0] == 0 and after.tolist() == [-1]
