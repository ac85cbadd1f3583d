"""Cached autoregressive generation for the GPT engine.

Prefill runs the engine's own forward over each prompt (flash attention) and
appends every layer's keys/values into a paged cache; each decode step then
processes one new token per active sequence: embedding -> per layer
LayerNorm -> QKV GEMM -> append K/V (paged_kv_append) -> paged decode
attention over the sequence's page chain -> projection GEMM (+residual) ->
LayerNorm -> GELU MLP GEMMs -> final LayerNorm -> LM head -> next token.
All layers share one page table (the pages of layer l live in layer l's
pool at the same page ids). Sequences can be forked (several samples of one
prompt share its pages; a step of samples of one prompt reads them once, a
step over several prompts reads each chain by itself), and `verify` feeds a few
drafted tokens per sequence at once and keeps those that the model confirms.

Reference parity: the reference generates with its (placeholder) GPT on the
CPU without a cache (scirs2-neural/src/models/architectures/gpt.rs); the
page management follows scirs2-neural/src/inference/block_manager.rs.
"""
from __future__ import annotations

from contextlib import contextmanager

import torch

from .. import _ext
from ..ops import kernels as K
from .kv_cache import BlockManager, BlockManagerConfig, InferenceError, KvPageConfig, KvPagePool
from .paged_attention import PagedAttentionConfig, PagedAttentionForward
from .speculative import verify_drafts


class GPTGenerator:
    def __init__(self, model, max_sequences: int = 16, max_len: int | None = None, block_size: int = 16,
                 num_pages: int | None = None):
        self.m = model
        cfg = model.cfg
        self.cfg = cfg
        self.L, self.H, self.hd, self.D = cfg.num_hidden_layers, cfg.num_attention_heads, cfg.head_dim, cfg.hidden_size
        max_len = max_len or cfg.max_position_embeddings
        pages_per_seq = (max_len + block_size - 1) // block_size
        num_pages = num_pages or max_sequences * pages_per_seq
        pc = KvPageConfig(block_size=block_size, num_heads=self.H, head_dim=self.hd)
        self.pools = [KvPagePool(num_pages, pc, model.device) for _ in range(self.L)]
        self.manager = BlockManager(self.pools[0], BlockManagerConfig(max_sequences, pages_per_seq), self.pools)
        self.attn = PagedAttentionForward(PagedAttentionConfig(self.H, self.hd))
        self.max_len = max_len
        self._next_id = 0
        self.last_token: dict[int, int] = {}

    # ----------------------------------------------------------- helpers
    def _append(self, l: int, rows, pos, k, v):
        dev = self.m.device
        mgr = self.manager
        if k.is_cuda:
            r = torch.tensor(rows, dtype=torch.int32).to(dev, non_blocking=True)
            p = torch.tensor(pos, dtype=torch.int32).to(dev, non_blocking=True)
            _ext.kernels().paged_kv_append(k.contiguous(), v.contiguous(), self.pools[l].k, self.pools[l].v,
                                           mgr.block_tables, r, p)
        else:
            bs = self.pools[0].config.block_size
            for i, (row, ps) in enumerate(zip(rows, pos)):
                pid = int(mgr._bt_host[row, ps // bs])
                self.pools[l].k[pid, ps % bs] = k[i]
                self.pools[l].v[pid, ps % bs] = v[i]

    @contextmanager
    def _undone(self, seq_ids: list[int], lens: list[int]):
        """Sequences that have grown go back to their lengths `lens` if the block does not end well."""
        try:
            yield
        except BaseException:
            for s, n in zip(seq_ids, lens):
                self.manager.truncate_sequence(s, n)
            raise

    @torch.no_grad()
    def _prefill(self, prompt: torch.Tensor) -> tuple[int, torch.Tensor]:
        """A new sequence with the prompt's tokens, without a pending one; its id and its last logits (fp32)."""
        m, H, hd = self.m, self.H, self.hd
        S = int(prompt.numel())
        assert 0 < S < self.max_len
        sid = self._next_id
        self._next_id += 1
        self.manager.allocate_sequence(sid)
        try:
            rows, pos = self.manager.reserve([sid], [S])
            self.manager.sync()
            tok = prompt.to(m.device).reshape(1, S)
            logits = m.logits(tok)  # runs every layer; keeps qkv per layer in the activations
            A = m._acts
            for l in range(self.L):
                qkv = A.qkv[l].view(S, 3, H, hd)
                self._append(l, rows, pos, qkv[:, 1], qkv[:, 2])
        except BaseException:  # no pages for the prompt, say: no half-made sequence stays behind
            self.manager.free_sequence(sid)
            raise
        return sid, logits[0, -1].float()

    # ----------------------------------------------------------- API
    @torch.no_grad()
    def add_sequence(self, prompt: torch.Tensor) -> int:
        """Prefill one prompt (1-D token tensor); returns the sequence id. The model's own choice (the
        largest logit) is the sequence's pending token."""
        sid, logits = self._prefill(prompt)
        self.last_token[sid] = int(torch.argmax(logits))
        return sid

    def fork(self, seq_id: int) -> int:
        """A copy of a sequence (its tokens and its pending one) that goes its own way from here. The
        two share their pages until one of them writes into one; a step whose sequences all begin with
        the same pages reads those once."""
        sid = self._next_id
        self.manager.fork_sequence(seq_id, sid)
        self._next_id += 1
        self.last_token[sid] = self.last_token[seq_id]
        return sid

    def _decode(self, toks, posn, rows, pos, attend) -> torch.Tensor:
        """Logits (fp32) of new tokens toks [n] at positions posn, whose keys and values go to the
        (row, position) pairs; attend(q [n, H, hd], pool) is the attention over the cache."""
        m, fp, cfg = self.m, self.m.fp, self.cfg
        H, hd, D = self.H, self.hd, self.D
        n = toks.numel()
        dev = m.device
        bf, f32 = torch.bfloat16, torch.float32
        x = (fp.w("wte")[toks].float() + fp.w("wpe")[posn].float()).to(bf).contiguous()
        ln = torch.empty(n, D, dtype=bf, device=dev)
        mu, rs = torch.empty(n, dtype=f32, device=dev), torch.empty(n, dtype=f32, device=dev)
        qkv = torch.empty(n, 3 * D, dtype=bf, device=dev)
        xm = torch.empty(n, D, dtype=bf, device=dev)
        h = torch.empty(n, cfg.intermediate_size, dtype=bf, device=dev)
        g = torch.empty(n, cfg.intermediate_size, dtype=bf, device=dev)
        eps = cfg.layer_norm_eps
        for l in range(self.L):
            p = f"h{l}."
            K.layernorm_fwd(x, fp.w(p + "ln_1.weight"), fp.w(p + "ln_1.bias"), ln, mu, rs, eps)
            K.gemm(ln, fp.w(p + "attn.c_attn.weight"), qkv, bias=fp.w(p + "attn.c_attn.bias"))
            q3 = qkv.view(n, 3, H, hd)
            self._append(l, rows, pos, q3[:, 1], q3[:, 2])
            att = attend(q3[:, 0], self.pools[l])
            K.gemm(att.reshape(n, D), fp.w(p + "attn.c_proj.weight"), xm, epi=K.EPI_RESID,
                   bias=fp.w(p + "attn.c_proj.bias"), aux=x)
            K.layernorm_fwd(xm, fp.w(p + "ln_2.weight"), fp.w(p + "ln_2.bias"), ln, mu, rs, eps)
            K.gemm(ln, fp.w(p + "mlp.c_fc.weight"), g, epi=K.EPI_BIAS_GELU, bias=fp.w(p + "mlp.c_fc.bias"), out2=h)
            x2 = torch.empty_like(x)
            K.gemm(g, fp.w(p + "mlp.c_proj.weight"), x2, epi=K.EPI_RESID, bias=fp.w(p + "mlp.c_proj.bias"), aux=xm)
            x = x2
        K.layernorm_fwd(x, fp.w("ln_f.weight"), fp.w("ln_f.bias"), ln, mu, rs, eps)
        logits = torch.empty(n, cfg.vocab_padded, dtype=bf, device=dev)
        K.gemm(ln, fp.w("wte"), logits)
        return logits[:, : cfg.vocab_size].float()

    @staticmethod
    def _draw(logits: torch.Tensor, temperature: float, generator=None) -> list[int]:
        """A token of each row of logits [n, vocab] at a temperature."""
        p = torch.softmax(logits / temperature, -1)
        # A row without a distribution is NaN throughout. On the GPU multinomial would find it by an assertion on
        # the device, which ends the process's use of it: such a row gets any weights, and no token.
        bad = torch.isnan(p[:, :1])
        t = torch.multinomial(p.masked_fill_(bad, 1.0), 1, generator=generator).masked_fill_(bad, -1).view(-1).tolist()
        if any(x < 0 for x in t):
            raise InferenceError("the model's probabilities hold no token to draw")
        return t

    def _cache_of(self, seq_ids: list[int]):
        """Tables and lengths of the batch, and the pages that all its chains begin with."""
        dev = self.m.device
        idx = torch.tensor([self.manager.row_of(s) for s in seq_ids], dtype=torch.long, device=dev)
        pages, shared = self.manager.shared_prefix(seq_ids) if len(seq_ids) > 1 else ([], 0)
        pages = torch.tensor(pages, dtype=torch.int32).to(dev) if shared else idx.new_empty(0, dtype=torch.int32)
        return (self.manager.block_tables[idx].contiguous(), self.manager.seq_lens[idx].contiguous(), pages, shared)

    @torch.no_grad()
    def step(self, seq_ids: list[int], temperature: float = 0.0, generator=None) -> list[int]:
        """Feed each sequence's pending token, return the next tokens."""
        n = len(seq_ids)
        dev = self.m.device
        toks = torch.tensor([self.last_token[s] for s in seq_ids], dtype=torch.long, device=dev)
        lens = [self.manager.seq_len(s) for s in seq_ids]
        posn = torch.tensor(lens, dtype=torch.long, device=dev)
        rows, pos = self.manager.reserve(seq_ids, [1] * n)
        with self._undone(seq_ids, lens):
            self.manager.sync()
            bt, sl, pages, shared = self._cache_of(seq_ids)

            def attend(q, pool):
                # Forked sequences: the pages they all begin with are read once. One shared page is enough: 2 to
                # 64 sequences of 40 to 1000 tokens, 12 heads of 64, 16 to 976 shared 11 to 73 us, else 20 to 214.
                if shared:
                    return self.attn.forward_shared_prefix(q, pool, bt, sl, pages, shared)
                return self.attn.forward_batch(q.contiguous(), pool, bt, sl)

            lg = self._decode(toks, posn, rows, pos, attend)
            if temperature > 0:
                out = self._draw(lg, temperature, generator)
            else:
                out = torch.argmax(lg, dim=-1).tolist()
        for s, t in zip(seq_ids, out):
            self.last_token[s] = t
        return out

    @torch.no_grad()
    def verify(self, seq_ids: list[int], drafts: list[list[int]], draft_probs: torch.Tensor | None = None,
               temperature: float = 0.0, uniforms: torch.Tensor | None = None, generator=None) -> list[list[int]]:
        """One step of speculative decoding: feed each sequence's pending token and its drafted ones
        (drafts[i], any number of them), keep the drafts that the model confirms, and return per
        sequence those and the token that follows, which becomes its pending one.

        draft_probs [B, n, vocab] (fp32, bf16 or fp16), n the largest number of drafts, holds the
        distributions that the drafts were drawn from (None: the draft is certain of them); uniforms
        fp32 [B, n + 1] the random numbers (default: drawn here); both on the model's device.
        Temperature 0 keeps the drafts that equal the model's own choice. The cache of rejected drafts
        is given back (speculative.verify_drafts). A call that raises leaves every sequence as it was."""
        B, dev, mgr = len(seq_ids), self.m.device, self.manager
        if len(drafts) != B:
            raise InferenceError("one list of drafts per sequence")
        if len(set(seq_ids)) < B:
            raise InferenceError("a sequence is verified once at a time")
        if not B:
            return []
        counts = [1 + len(d) for d in drafts]
        Q = max(counts)
        lens = [mgr.seq_len(s) for s in seq_ids]
        if any(a + c > self.cfg.max_position_embeddings for a, c in zip(lens, counts)):
            raise InferenceError("sequence exceeds the model's positions")
        fed = [t for s, d in zip(seq_ids, drafts) for t in (self.last_token[s], *d)]
        if any(not 0 <= t < self.cfg.vocab_size for t in fed):
            raise InferenceError("drafted token outside the vocabulary")
        place = self.pools[0].k.device
        if draft_probs is not None:
            if draft_probs.shape != (B, Q - 1, self.cfg.vocab_size):
                raise InferenceError(f"draft_probs must be [{B}, {Q - 1}, {self.cfg.vocab_size}]")
            if draft_probs.dtype not in (torch.float32, torch.bfloat16, torch.float16) or draft_probs.device != place:
                raise InferenceError(f"draft_probs must be fp32, bf16 or fp16 on {place}")
        if uniforms is not None:
            if uniforms.shape != (B, Q):
                raise InferenceError(f"uniforms must be [{B}, {Q}]")
            if uniforms.dtype != torch.float32 or uniforms.device != place:
                raise InferenceError(f"uniforms must be fp32 on {place}")
        toks = torch.tensor(fed, dtype=torch.long, device=dev)
        posn = torch.tensor([a + i for a, c in zip(lens, counts) for i in range(c)], dtype=torch.long, device=dev)
        at = torch.tensor([b * Q + i for b, c in enumerate(counts) for i in range(c)], dtype=torch.long, device=dev)
        rows, pos = mgr.reserve(seq_ids, counts)
        with self._undone(seq_ids, lens):
            mgr.sync()
            bt, sl, pages, shared = self._cache_of(seq_ids)
            ql = torch.tensor(counts, dtype=torch.int32, device=dev)

            def attend(q, pool):
                q4 = torch.zeros(B * Q, self.H, self.hd, dtype=q.dtype, device=dev)
                q4[at] = q
                o = self.attn.forward_shared_prefix(q4.view(B, Q, self.H, self.hd), pool, bt, sl, pages, shared, ql)
                return o.view(B * Q, self.H, self.hd)[at]

            lg = self._decode(toks, posn, rows, pos, attend)
            if temperature > 0:
                p = torch.softmax(lg / temperature, -1)
            else:
                best = torch.argmax(lg, -1, keepdim=True)  # (a NaN, where the row holds one: no token then)
                p = torch.zeros_like(lg).scatter_(1, best, 1.0 - torch.isnan(lg.gather(1, best)).float())
            target = torch.zeros(B * Q, p.shape[1], device=dev)
            target[at] = p
            dt = torch.tensor([list(d) + [-1] * (Q - 1 - len(d)) for d in drafts], dtype=torch.long)
            if uniforms is None:
                uniforms = torch.rand(B, Q, device=dev, generator=generator)
            if draft_probs is not None:  # (a wider type holds the same values)
                draft_probs = draft_probs.float()
            kept, new = verify_drafts(target.view(B, Q, -1), draft_probs, dt.view(B, Q - 1).to(dev), uniforms,
                                      torch.tensor([c - 1 for c in counts], dtype=torch.int32, device=dev))
            out = [t[: k + 1] for k, t in zip(kept.tolist(), new.tolist())]
            if any(t[-1] < 0 for t in out):  # logits that are no numbers
                raise InferenceError("the model's probabilities hold no token to draw")
        for s, a, t in zip(seq_ids, lens, out):
            mgr.truncate_sequence(s, a + len(t))
            self.last_token[s] = t[-1]
        return out

    def generate(self, prompts: list[torch.Tensor], max_new_tokens: int, temperature: float = 0.0,
                 num_samples: int = 1) -> list[list[int]]:
        """Greedy (temperature 0) or sampled continuation of every prompt, num_samples of each (prompt
        by prompt; the prompt is processed once and forked). At a temperature every token of every
        sample is drawn, the first one too."""
        if num_samples < 1:
            raise ValueError("num_samples must be at least 1")
        ids = []
        try:
            for p in prompts:
                sid, logits = self._prefill(p)
                ids.append(sid)
                if temperature > 0:
                    first = self._draw(logits.expand(num_samples, -1), temperature)
                else:
                    first = [int(torch.argmax(logits))] * num_samples
                self.last_token[sid] = first[0]
                for t in first[1:]:
                    ids.append(self.fork(sid))
                    self.last_token[ids[-1]] = t
            outs = {s: [self.last_token[s]] for s in ids}
            for _ in range(max_new_tokens - 1):
                for s, t in zip(ids, self.step(ids, temperature)):
                    outs[s].append(t)
        finally:  # no row or page left for a sample, say: those that were made are given back
            for s in ids:
                self.release(s)
        return [outs[s] for s in ids]

    def release(self, seq_id: int):
        self.manager.free_sequence(seq_id)
        self.last_token.pop(seq_id, None)
