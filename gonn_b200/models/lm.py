"""Language models composed from the nn layers.

``TransformerLM``: token + position embeddings, N pre-LayerNorm encoder layers
with causal self-attention and a GELU feed-forward, final LayerNorm, untied
vocabulary projection.  ``GPT``: decoder-only blocks with RMSNorm, causal
attention and a GELU feed-forward.  Parameter names follow the reference's
naming contract for the layers they reuse (``layers.N.attn.qproj.weight``, ...).

``GPT(rotary=...)`` has rotary positions in place of the table of learned ones.  ``GPT.Generate`` writes on token by token from a paged
cache (``GPT.Step``); several samples of one prompt share the prompt's pages.
"""
from __future__ import annotations

import torch

from ..nn import block as _block
from ..nn.activation import GELU
from ..nn.attention import MultiHeadAttention
from ..nn.cache import KVCache, RotaryEmbedding
from ..nn.embedding import Embedding
from ..nn.linear import Linear
from ..nn.module import Module, ModuleList
from ..nn.norm import LayerNorm, RMSNorm
from ..nn.transformer import ENCODER_FORWARD, TransformerEncoderLayer
from ..ops.elementwise import binary as _binary
from ..ops.linear import feed_forward as _feed_forward
from ..ops.softmax import cross_entropy


class TransformerLM(Module):
    def __init__(self, vocab: int = 32000, d_model: int = 768, n_layers: int = 12, n_heads: int = 12,
                 d_ff: int = 3072, max_seq: int = 1024, *, dtype=torch.float32, device=None):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.vocab, self.d_model, self.max_seq = vocab, d_model, max_seq
        self.tok = Embedding(vocab, d_model, **kw)
        self.pos = Embedding(max_seq, d_model, **kw)
        self.layers = ModuleList([
            TransformerEncoderLayer(d_model, n_heads, d_ff, pre_norm=True, activation=GELU(), causal=True, **kw)
            for _ in range(n_layers)])
        self.norm = LayerNorm(d_model, **kw)
        self.head = Linear(d_model, vocab, bias=False, **kw)
        with torch.no_grad():
            self.tok.weight.mul_(0.02)
            self.pos.weight.mul_(0.02)

    def forward(self, ids):
        B, S = ids.shape
        pos = torch.arange(S, device=ids.device)
        x = _binary("add", self.tok(ids), self.pos(pos)[None])
        x = _block.chain(x, self.layers, TransformerEncoderLayer, ENCODER_FORWARD)
        return self.head(self.norm(x))

    def loss(self, ids, targets):
        """Mean next-token cross-entropy; the logits' gradient overwrites the logits."""
        logits = self.forward(ids)
        return cross_entropy(logits.reshape(-1, self.vocab), targets.reshape(-1), inplace_backward=True,
                             consume_logits=True)


class GPTBlock(Module):
    def __init__(self, d_model: int, n_heads: int, d_ff: int, *, rotary=None, dtype=torch.float32, device=None):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.norm1 = RMSNorm(d_model, **kw)
        self.attn = MultiHeadAttention(d_model, n_heads, rotary=rotary, **kw)
        self.norm2 = RMSNorm(d_model, **kw)
        self.ff1 = Linear(d_model, d_ff, True, **kw)
        self.ff2 = Linear(d_ff, d_model, True, **kw)

    def _parts(self):
        m = self._modules
        return m["attn"], m["norm1"], m["norm2"], m["ff1"], m["ff2"], "gelu", True, True

    def forward(self, x):
        if not torch.is_grad_enabled() and type(self) is GPTBlock:
            y = _block.evaluate(x, *self._parts())
            if y is not None:
                return y
        f1 = self.norm1.fork(x, self.attn.outproj.bias) if torch.is_grad_enabled() else None
        if f1 is not None:
            x = self.attn(f1[0], f1[0], f1[0], True, residual=f1[1], out_bias_grad=False)
        else:
            n = self.norm1(x)
            x = self.attn(n, n, n, True, residual=x)
        f2 = self.norm2.fork(x, self.ff2.bias) if torch.is_grad_enabled() else None
        if f2 is not None:
            return _feed_forward(f2[0], self.ff1.weight, self.ff1.bias, self.ff2.weight, self.ff2.bias,
                                 "gelu", f2[1], False)
        return _feed_forward(self.norm2(x), self.ff1.weight, self.ff1.bias, self.ff2.weight, self.ff2.bias,
                             "gelu", x)


    def Step(self, x, cache, table, lengths, counts=None, shared_pages: int = 0):
        """New tokens x (B, T, d_model) behind those in the cache (see ``MultiHeadAttention.ForwardCached``)."""
        x = self.attn.ForwardCached(self.norm1(x), cache, table, lengths, counts, shared_pages, residual=x)
        return _feed_forward(self.norm2(x), self.ff1.weight, self.ff1.bias, self.ff2.weight, self.ff2.bias,
                             "gelu", x)


GPT_FORWARD = GPTBlock.forward


class GPT(Module):
    """Decoder-only LM: 24 x (2048, 16 heads, 8192) with vocab 50304 is the 1.3 B config."""

    def __init__(self, vocab: int = 50304, d_model: int = 2048, n_layers: int = 24, n_heads: int = 16,
                 d_ff: int = 8192, max_seq: int = 2048, *, rotary=None, dtype=torch.float32, device=None):
        """``rotary``: True, or the options of a ``RotaryEmbedding`` (dim: the head size), for rotary instead of learned positions."""
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.vocab, self.d_model, self.max_seq = vocab, d_model, max_seq
        self.tok = Embedding(vocab, d_model, **kw)
        if rotary is None or rotary is False:
            rope, self.pos = None, Embedding(max_seq, d_model, **kw)
        else:
            rope, self.pos = RotaryEmbedding(**{"dim": d_model // n_heads, **({} if rotary is True else rotary)}, device=device), None
        self.layers = ModuleList([GPTBlock(d_model, n_heads, d_ff, rotary=rope, **kw) for _ in range(n_layers)])
        self.norm = RMSNorm(d_model, **kw)
        self.head = Linear(d_model, vocab, bias=False, **kw)
        with torch.no_grad():
            self.tok.weight.mul_(0.02)
            if self.pos is not None:
                self.pos.weight.mul_(0.02)

    def forward(self, ids):
        B, S = ids.shape
        x = self.tok(ids)
        if self.pos is not None:
            x = _binary("add", x, self.pos(torch.arange(S, device=ids.device))[None])
        x = _block.chain(x, self.layers, GPTBlock, GPT_FORWARD)
        return self.head(self.norm(x))

    def loss(self, ids, targets):
        logits = self.forward(ids)
        return cross_entropy(logits.reshape(-1, self.vocab), targets.reshape(-1), inplace_backward=True,
                             consume_logits=True)

    def Caches(self, pages: int, page_size: int = 64):
        """A ``KVCache`` for every block, all with the same pages."""
        w, a = self.tok.weight, self.layers[0].attn
        return [KVCache(pages, page_size, a.num_heads, a.head_dim, dtype=w.dtype, device=w.device) for _ in self.layers]

    def Step(self, ids, caches, table, lengths, counts=None, shared_pages: int = 0):
        """Logits (B, T, vocab) of new tokens ids (B, T) behind the ``lengths`` positions of their sequences that the caches hold, which
        take the new ones up (see ``KVCache`` for table, lengths, counts and shared_pages).  For evaluation: under torch.no_grad()."""
        x = self.tok(ids)
        if self.pos is not None:
            token = torch.arange(ids.shape[1], device=ids.device)
            at = lengths.long()[:, None] + token
            if counts is not None:               # tokens that do not count may lie behind the last position
                at = torch.where(token < counts[:, None], at, 0)
            x = _binary("add", x, self.pos(at))
        for block, cache in zip(self.layers, caches):
            x = block.Step(x, cache, table, lengths, counts, shared_pages)
        return self.head(self.norm(x))

    @torch.no_grad()
    def Generate(self, ids, new_tokens: int, samples: int = 1, temperature: float = 0.0, page_size: int = 64):
        """ids (B, S) with ``new_tokens`` more each: the most likely one (temperature 0), or drawn.  ``samples`` > 1: that many continuations of
        one prompt (B = 1), whose pages they share, as (samples, S + new_tokens)."""
        B, S = ids.shape
        if S < 1 or new_tokens < 0 or samples < 1 or (samples > 1 and B != 1):
            raise ValueError("GPT.Generate: a prompt of at least one token, new_tokens >= 0, and one prompt for several samples")
        if self.pos is not None and S + new_tokens > self.max_seq:
            raise ValueError(f"GPT.Generate: {S + new_tokens} positions, the model has {self.max_seq}")
        if new_tokens == 0:
            return ids.expand(samples, S).clone() if samples > 1 else ids.clone()
        shared = S // page_size if samples > 1 else 0
        rows, columns = max(B, samples), -(-(S + new_tokens) // page_size)
        own = columns - shared
        table = torch.empty(rows, columns, dtype=torch.int32)
        table[:, :shared] = torch.arange(shared)
        table[:, shared:] = shared + torch.arange(rows * own).view(rows, own)
        table = table.to(ids.device)
        caches = self.Caches(shared + rows * own, page_size)
        lengths = torch.zeros(rows, dtype=torch.int32, device=ids.device)
        logits = self.Step(ids, caches, table[:B], lengths[:B])[:, -1:]
        if samples > 1:
            if S % page_size:                    # the prompt's last page is begun: every sample goes on with its own copy
                for c in caches:
                    for t in (c.Keys, c.Values):
                        t[shared + own::own] = t[shared].clone()
            ids, logits = ids.expand(samples, S), logits.expand(samples, 1, -1)
        lengths += S
        out = [ids]
        for i in range(new_tokens):
            z = logits[:, -1].float()
            if temperature > 0:
                new = torch.multinomial(torch.softmax(z / temperature, -1), 1)
            else:
                new = z.argmax(-1, keepdim=True)
            out.append(new)
            if i + 1 < new_tokens:
                logits = self.Step(new, caches, table, lengths, shared_pages=shared)
                lengths += 1
        return torch.cat(out, 1)
