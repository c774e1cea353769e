"""GPT training step with Co-ALiBi attention: the caller of the attention hot path.

The reference has no model code; its benchmark configs name this one (12 layers,
d_model 768, 12 heads of 64, no positional embeddings, vocab 50304, B=8, S=1024,
bf16 autocast, AdamW, one fwd+bwd+step).  Positions enter only through the
Co-ALiBi penalty of ``co_alibi_attention`` (the 12-head slope table uses the
non-power-of-two branch of ``_get_coalibi_slopes``).

The block is a standard pre-norm transformer block: LayerNorm, fused QKV
projection, causal Co-ALiBi attention, output projection, residual; LayerNorm,
GELU MLP (4x), residual.  The LM head is tied to the token embedding.

``attention`` is injectable so tests can run the same model on the CPU with a
reference attention; the default is the native ``co_alibi_attention``.

Serving: ``GPT.prefill`` and ``GPT.extend`` run new tokens over a ``PagedCache`` and each other, ``PagedCache.accept``
keeps their keys and values, ``GPT.generate`` samples with them, and ``GPT.speculate`` checks a tree of drafts.  These
call the native operators (co_alibi_attn/serving.py), on the GPU only.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable

import torch
import torch.nn as nn
import torch.nn.functional as F

from .co_alibi_attn import co_alibi_attention, co_alibi_attention_qkv
from .serving import co_alibi_cache_append, co_alibi_decode_tree, co_alibi_sample


@dataclass(frozen=True)
class GPTConfig:
    n_layer: int = 12
    n_head: int = 12
    d_model: int = 768
    vocab: int = 50304
    mlp_ratio: int = 4
    bias_max: float = 8.0


AttentionFn = Callable[..., torch.Tensor]


class PagedCache:
    """Every layer's keys and values of a batch of sequences, in pages under one block table.

    ``capacity`` rows per sequence, all empty at first.  ``dtype`` is the one the model's projections have (the
    weights' type, or autocast's).  A forward over the cache leaves its new keys and values in ``new``, one
    (k, v) per layer; ``accept`` writes them.

    A step with ``accept`` in it may be captured and replayed.  A replay cannot raise: rows without room are dropped
    and the lengths stay at the capacity.  The host sees no replay, so that from the capture on ``room_for`` reads the lengths
    from the device (it waits for them): call it between replays to be told of a cache that fills up.
    """

    def __init__(self, cfg: GPTConfig, batch: int, capacity: int, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda", page_size: int = 64):
        blocks = -(-capacity // page_size)
        self.capacity = blocks * page_size
        shape = (batch * blocks, cfg.n_head, page_size, cfg.d_model // cfg.n_head)
        self.layers = [(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
                       for _ in range(cfg.n_layer)]
        self.block_table = torch.arange(batch * blocks, dtype=torch.int32, device=device).view(batch, blocks)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.bound = 0  # no sequence is longer; known without reading the device, but for replays of a captured accept
        self.captured = False
        self.new: list[tuple[torch.Tensor, torch.Tensor]] = []

    def _capturing(self) -> bool:
        return self.seq_lens.is_cuda and torch.cuda.is_current_stream_capturing()

    def room_for(self, tokens: int) -> None:
        """Raises ValueError where a sequence has no room for this many more rows (not in a capture: see above)."""
        if self._capturing():
            return
        # The bound counts every row as accepted, and no replayed one: look before refusing, or before relying on it.
        if self.captured or self.bound + tokens > self.capacity:
            self.bound = int(self.seq_lens.max())
        if self.bound + tokens > self.capacity:
            raise ValueError(f"{tokens} more rows behind {self.bound} do not fit a cache of {self.capacity}")

    def accept(self, rows: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
        """Keeps the last forward's new rows: all, the first counts[b], or the rows[b, :counts[b]] (a path of a tree).

        All rows have to fit (ValueError, but in a capture); of ``counts``, which are on the device, what fits is kept.
        """
        if not self.new:
            raise ValueError("no new keys and values: run a forward over this cache first")
        n = self.new[0][0].shape[2] if rows is None else rows.shape[1]
        if counts is None:
            self.room_for(n)
        for (k_cache, v_cache), (k, v) in zip(self.layers, self.new):
            co_alibi_cache_append(k, v, k_cache, v_cache, self.seq_lens, self.block_table, rows=rows, counts=counts)
        if self._capturing():
            self.captured = True
        if counts is not None:
            self.seq_lens += torch.minimum(counts.clamp(0, n), self.capacity - self.seq_lens)
        elif self.captured:
            self.seq_lens.add_(n).clamp_(max=self.capacity)
        else:
            self.seq_lens += n
        self.bound = min(self.bound + n, self.capacity)
        self.new = []


class CausalCoALiBiAttention(nn.Module):
    def __init__(self, cfg: GPTConfig, attention: AttentionFn):
        super().__init__()
        self.n_head = cfg.n_head
        self.head_dim = cfg.d_model // cfg.n_head
        self.bias_max = cfg.bias_max
        self.qkv = nn.Linear(cfg.d_model, 3 * cfg.d_model, bias=False)
        self.proj = nn.Linear(cfg.d_model, cfg.d_model, bias=False)
        self.attention = attention

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, S, C = x.shape
        qkv = self.qkv(x).view(B, S, 3, self.n_head, self.head_dim)
        if self.attention is co_alibi_attention and qkv.is_cuda:
            # The same attention on the packed projection: no copies of its parts, and one packed
            # gradient in place of three that autograd would zero-fill and add.
            return self.proj(co_alibi_attention_qkv(qkv, causal=True, bias_max=self.bias_max).reshape(B, S, C))
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))  # (B, H, S, D) views
        y = self.attention(q, k, v, causal=True, bias_max=self.bias_max)
        return self.proj(y.transpose(1, 2).reshape(B, S, C))

    def over_cache(self, x: torch.Tensor, cache: PagedCache, layer: int, parents: torch.Tensor | None,
                   prefill: bool) -> tuple[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
        """The attention of new tokens (B, T, C) over one layer of the cache, and their (k, v)."""
        B, T, C = x.shape
        qkv = self.qkv(x).view(B, T, 3, self.n_head, self.head_dim)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        if prefill:
            y = co_alibi_attention_qkv(qkv, causal=True, bias_max=self.bias_max)
        else:
            y = co_alibi_decode_tree(q, k, v, *cache.layers[layer], seq_len=cache.seq_lens, parents=parents,
                                     block_table=cache.block_table, bias_max=self.bias_max).transpose(1, 2)
        return self.proj(y.reshape(B, T, C)), (k, v)


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig, attention: AttentionFn):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.d_model)
        self.attn = CausalCoALiBiAttention(cfg, attention)
        self.ln2 = nn.LayerNorm(cfg.d_model)
        self.fc = nn.Linear(cfg.d_model, cfg.mlp_ratio * cfg.d_model)
        self.out = nn.Linear(cfg.mlp_ratio * cfg.d_model, cfg.d_model)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.mlp(x + self.attn(self.ln1(x)))

    def mlp(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))


class GPT(nn.Module):
    def __init__(self, cfg: GPTConfig = GPTConfig(), attention: AttentionFn = co_alibi_attention):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab, cfg.d_model)
        self.blocks = nn.ModuleList(Block(cfg, attention) for _ in range(cfg.n_layer))
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.apply(self._init)
        # GPT-2 style scaled init of the residual projections.
        for name, p in self.named_parameters():
            if name.endswith("attn.proj.weight") or name.endswith("out.weight"):
                nn.init.normal_(p, mean=0.0, std=0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init(m: nn.Module) -> None:
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)

    def forward(self, idx: torch.Tensor, targets: torch.Tensor | None = None):
        x = self.wte(idx)
        for blk in self.blocks:
            x = blk(x)
        logits = F.linear(self.ln_f(x), self.wte.weight)  # tied LM head
        if targets is None:
            return logits
        loss = F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.view(-1))
        return logits, loss

    def _over_cache(self, idx: torch.Tensor, cache: PagedCache, parents=None, prefill=False) -> torch.Tensor:
        cache.new = []
        new: list[tuple[torch.Tensor, torch.Tensor]] = []
        x = self.wte(idx.clamp(min=0))  # -1, co_alibi_sample's for a row without a token, is no row of the embedding
        for i, blk in enumerate(self.blocks):
            y, kv = blk.attn.over_cache(blk.ln1(x), cache, i, parents, prefill)
            x = blk.mlp(x + y)
            new.append(kv)
        cache.new = new  # all layers' or none
        return self.ln_f(x)

    @torch.no_grad()
    def prefill(self, idx: torch.Tensor, cache: PagedCache, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Puts prompts (B, S) into an empty cache; returns the logits (B, vocab) behind each one's last token.

        ``lengths``: integer tensor (B,) with values in [1, S], others are clamped: sequence b is idx[b, :lengths[b]], the
        rest padding.
        """
        B, S = idx.shape
        if S < 1:
            raise ValueError("a prompt needs at least one token")
        cache.room_for(0)  # the bound, where replays have moved the lengths
        if cache.bound != 0:
            raise ValueError("prefill needs an empty cache")
        cache.room_for(S)
        lengths = None if lengths is None else lengths.clamp(1, S)
        h = self._over_cache(idx, cache, prefill=True)
        cache.accept(counts=lengths)
        h = h[:, -1] if lengths is None else h[torch.arange(B, device=h.device), lengths.long() - 1]
        return F.linear(h, self.wte.weight)

    @torch.no_grad()
    def extend(self, idx: torch.Tensor, cache: PagedCache, parents: torch.Tensor | None = None) -> torch.Tensor:
        """Logits (B, T, vocab) behind each of T <= 64 new tokens idx (B, T), a chain or the tree of ``parents``.

        The cache's rows stay as they are; ``cache.accept`` keeps the new ones.
        """
        return F.linear(self._over_cache(idx, cache, parents), self.wte.weight)

    @torch.no_grad()
    def generate(self, idx: torch.Tensor, lengths: torch.Tensor | None, uniforms: torch.Tensor, cache: PagedCache,
                 **sampling) -> torch.Tensor:
        """Tokens (B, n) that follow the prompts (as for ``prefill``), one per uniform number of ``uniforms`` (B, n).

        ``sampling``: the settings of ``co_alibi_sample``.  The last token is not in the cache.  A sequence for which no
        token can be drawn (logits with a NaN) has -1 there and from there on.
        """
        logits = self.prefill(idx, cache, lengths)
        out = torch.empty(uniforms.shape, dtype=torch.long, device=idx.device)
        for i in range(uniforms.shape[1]):
            if i > 0:
                cache.room_for(1)
                logits = self.extend(out[:, i - 1:i], cache)[:, 0]
                cache.accept()
            out[:, i] = co_alibi_sample(logits, uniforms[:, i], **sampling)
        return out.masked_fill_((out < 0).cumsum(1) > 0, -1)

    @torch.no_grad()
    def speculate(self, idx: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor, cache: PagedCache, **sampling):
        """One step over a tree of drafts; returns (rows (B, T), counts (B,), next tokens (B,)).

        idx, parents: (B, T).  Node 0 is the sequence's last token, which the cache does not hold yet, with parent -1; the
        others are drafts.  Behind every node one token is drawn with that node's number of ``uniforms`` (B, T).  A
        draft is accepted when its parent is and it is the token drawn there (the first of equal ones), so what
        is accepted, idx[b, rows[b, 1:counts[b]]], and the next token, drawn behind it, are what drawing token by token
        gives with those numbers.  The cache keeps the accepted rows; of a path that it has no room for, as many as fit are
        accepted (node 0 has to fit: ValueError).
        """
        B, T = idx.shape
        cache.room_for(1)
        logits = self.extend(idx, cache, parents)
        drawn = co_alibi_sample(logits.reshape(B * T, -1), uniforms.reshape(B * T), **sampling).view(B, T)
        node = torch.arange(T, device=idx.device)
        up = parents.long().clamp(0, T - 1)
        ok = (idx == drawn.gather(1, up)) & (idx >= 0) & (parents >= 0) & (parents < node)
        # (Of nodes that are there: one whose parent comes after it is absent.)
        same = (parents[:, :, None] == parents[:, None]) & (idx[:, :, None] == idx[:, None])
        ok &= ~(same & (node < node[:, None]) & ok[:, None]).any(2)
        ok[:, 0] = True
        up[:, 0] = 0
        for _ in range(T.bit_length()):  # accepted: so are 1, 2, 4, ... ancestors
            ok &= ok.gather(1, up)
            up = up.gather(1, up)
        # What is accepted is one path, in the nodes' order: what fits is its beginning.
        counts = torch.minimum(ok.sum(1, dtype=torch.int32), cache.capacity - cache.seq_lens)
        rows = torch.where(ok, node, T).sort(1).values.int()
        cache.accept(rows, counts)
        last = rows.gather(1, counts[:, None].long().clamp(min=1) - 1).long()
        return rows, counts, drawn.gather(1, last)[:, 0]

    def n_params(self) -> int:
        return sum(p.numel() for p in self.parameters())


def make_optimizer(model: GPT, lr: float = 6e-4, weight_decay: float = 0.1) -> torch.optim.Optimizer:
    """AdamW with weight decay on matrices only (embeddings and linear weights)."""
    decay = [p for p in model.parameters() if p.dim() >= 2]
    no_decay = [p for p in model.parameters() if p.dim() < 2]
    groups = [{"params": decay, "weight_decay": weight_decay}, {"params": no_decay, "weight_decay": 0.0}]
    return torch.optim.AdamW(groups, lr=lr, betas=(0.9, 0.95), eps=1e-8)


def synthetic_batch(cfg: GPTConfig, batch: int, seq: int, seed: int = 0, device="cpu"):
    """Uniform-random token ids (inputs and next-token targets), drawn on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, cfg.vocab, (batch, seq + 1), generator=gen)
    return tok[:, :-1].contiguous().to(device), tok[:, 1:].contiguous().to(device)


def train_step(model: GPT, opt: torch.optim.Optimizer, idx: torch.Tensor, targets: torch.Tensor,
               autocast_dtype: torch.dtype | None = torch.bfloat16) -> torch.Tensor:
    """One forward + backward + AdamW step; returns the (detached) loss."""
    opt.zero_grad(set_to_none=True)
    if autocast_dtype is None:
        _, loss = model(idx, targets)
    else:
        with torch.autocast(device_type=idx.device.type, dtype=autocast_dtype):
            _, loss = model(idx, targets)
    loss.backward()
    opt.step()
    return loss.detach()
