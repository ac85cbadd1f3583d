"""Single-query (decode) attention over paged KV caches.

:class:`PagedAttentionForward` computes, for every active sequence, the
attention of its newest query ([H, HD]) over the sequence's whole page chain,
with grouped-query heads (H query heads over Hkv cached heads). On the GPU
this is the split-key decode kernel of scirs_b200/csrc/paged_attention.cu
(bandwidth-bound: each cached K/V byte is read once per sequence and KV head)
followed by a combine kernel; on the CPU a PyTorch restatement.

:meth:`PagedAttentionForward.forward_shared_prefix` is the same for a batch
whose sequences begin with the same tokens (forks of one prompt, requests
behind one system prompt) and for several new tokens a sequence (drafted
tokens to be scored): the prefix is read once for the whole batch
(scirs_b200/csrc/prefix_attention.cu).

Reference parity: scirs2-neural/src/inference/paged_attention.rs:37-283
(PagedAttentionConfig, PagedAttentionForward::forward(query, page_chain,
pool)).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _ext
from ..ops import kernels as K
from .kv_cache import BlockManager, InferenceError, KvPagePool


@dataclass
class PagedAttentionConfig:
    num_heads: int = 8
    head_dim: int = 64
    scale: float | None = None
    tokens_per_split: int = 512


class PagedAttentionForward:
    def __init__(self, config: PagedAttentionConfig):
        self.config = config
        self._scratch = {}

    def _scale(self):
        c = self.config
        return c.scale if c.scale is not None else c.head_dim ** -0.5

    def forward(self, query: torch.Tensor, page_chain: list[int], pool: KvPagePool, seq_len: int | None = None):
        """One sequence: query [H, HD], its page chain, and (optionally) its
        length in tokens (default: the whole chain)."""
        bs = pool.config.block_size
        n = seq_len if seq_len is not None else len(page_chain) * bs
        if query.shape != (self.config.num_heads, self.config.head_dim):
            raise InferenceError("query shape does not match the configuration")
        bt = torch.tensor([page_chain], dtype=torch.int32, device=pool.device)
        lens = torch.tensor([n], dtype=torch.int32, device=pool.device)
        return self.forward_batch(query.reshape(1, *query.shape), pool, bt, lens)[0]

    def forward_batch(self, q: torch.Tensor, pool: KvPagePool, block_tables: torch.Tensor, seq_lens: torch.Tensor):
        """q [B, H, HD]; block_tables [B, max_pages] int32; seq_lens [B] int32."""
        B, H, HD = q.shape
        if q.is_cuda:
            c = self.config
            span = block_tables.shape[1] * pool.config.block_size
            splits = max(1, (span + c.tokens_per_split - 1) // c.tokens_per_split)
            key = (B, H, HD, splits)
            if key not in self._scratch:
                self._scratch = {key: (torch.empty(B, H, splits, HD, device=q.device),
                                       torch.empty(B, H, splits, 2, device=q.device))}
            po, pml = self._scratch[key]
            out = torch.empty(B, H, HD, dtype=torch.bfloat16, device=q.device)
            _ext.kernels().paged_attention_decode(q.to(torch.bfloat16).contiguous(), pool.k, pool.v,
                                                  block_tables.contiguous(), seq_lens.contiguous(), out, po, pml,
                                                  c.tokens_per_split, self._scale())
            return out
        return paged_attention_reference(q, pool, block_tables, seq_lens, self._scale())

    def forward_shared_prefix(self, q: torch.Tensor, pool: KvPagePool, block_tables: torch.Tensor,
                              seq_lens: torch.Tensor, prefix_pages: torch.Tensor, prefix_len: int,
                              q_lens: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the newest tokens of a batch whose first ``prefix_len`` tokens are the same.

        q [B, H, HD], or [B, Q, H, HD] for up to Q tokens a sequence; block_tables int32
        [B, max_pages], each sequence's whole chain; seq_lens int32 [B], its tokens with the newest
        ones; prefix_pages int32, the pages of the prefix (it may end inside one); q_lens int32 [B],
        how many of the Q queries a sequence has (default: all). Query t of a sequence stands at
        position ``seq_len - q_len + t`` and sees the keys up to there. Rows past q_len, and
        sequences of length 0, give zeros; a sequence with a query inside the prefix is read through
        its own chain from the first key on. Every head_dim that is a multiple of 8 up to 128, any
        number of query heads per cached head, any page size. bf16; the softmax and the sums are
        kept in fp32. A captured graph keeps prefix_len, and reads the tables and lengths anew.
        A page id outside of the pool is refused on the CPU; on the GPU its keys are left out, and the
        next check_status raises.
        """
        c, n = pool.config, self.config
        if q.dim() not in (3, 4) or q.shape[-2] != n.num_heads or q.shape[-1] != n.head_dim:
            raise InferenceError("query shape does not match the configuration")
        if n.num_heads % c.num_heads or n.head_dim != c.head_dim:
            raise InferenceError("the pool's heads do not match the configuration")
        scale = self._scale()
        if not 0.0 < scale < float("inf"):
            raise InferenceError("scale must be positive and finite")
        if prefix_len < 0 or prefix_len > min(prefix_pages.numel(), block_tables.shape[-1]) * c.block_size:
            raise InferenceError("prefix_len is longer than the prefix's pages or a chain")
        if q.is_cuda:
            if q.dtype != torch.bfloat16:
                q = q.to(torch.bfloat16)
            out, launches = _ext.kernels().paged_prefix_attention(q, pool.k, pool.v, block_tables, seq_lens,
                                                                  prefix_pages, int(prefix_len), q_lens, scale)
            K._count(launches)
            return out
        q4 = q.unsqueeze(1) if q.dim() == 3 else q
        out = shared_prefix_attention_reference(q4, pool, block_tables, seq_lens, prefix_pages, prefix_len, q_lens,
                                                scale)
        return out.reshape(q.shape)

    def forward_manager(self, q: torch.Tensor, manager: BlockManager, seq_ids: list[int]):
        """Decode attention for the given sequences of a BlockManager."""
        manager.sync()
        rows = torch.tensor([manager.row_of(s) for s in seq_ids], dtype=torch.long, device=manager.block_tables.device)
        return self.forward_batch(q, manager.pool, manager.block_tables[rows].contiguous(),
                                  manager.seq_lens[rows].contiguous())

    def forward_manager_shared(self, q: torch.Tensor, manager: BlockManager, seq_ids: list[int],
                               q_lens: torch.Tensor | None = None):
        """forward_shared_prefix for sequences of a BlockManager, over the pages that they share. The
        prefix ends where the first of the queries stands: pages may be shared up to the newest token
        (forks that have not been written to, a single sequence), and a sequence with a query inside the
        prefix would be read by itself."""
        manager.sync()
        dev = manager.block_tables.device
        pages, n = manager.shared_prefix(seq_ids)
        queries = q.shape[1] if q.dim() == 4 else 1
        n = max(0, min([n] + [manager.seq_len(s) - queries + 1 for s in seq_ids]))
        rows = torch.tensor([manager.row_of(s) for s in seq_ids], dtype=torch.long, device=dev)
        return self.forward_shared_prefix(q, manager.pool, manager.block_tables[rows], manager.seq_lens[rows],
                                          torch.tensor(pages, dtype=torch.int32, device=dev), n, q_lens)


def shared_prefix_attention_reference(q, pool: KvPagePool, block_tables, seq_lens, prefix_pages, prefix_len, q_lens,
                                      scale):
    """fp32 PyTorch restatement of forward_shared_prefix (oracle); q [B, Q, H, HD]."""
    B, Q, H, HD = q.shape
    Hkv, bs = pool.config.num_heads, pool.config.block_size
    G = H // Hkv
    out = torch.zeros(B, Q, H, HD, dtype=torch.bfloat16, device=q.device)
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), block_tables.shape[1] * bs)
        ql = Q if q_lens is None else min(max(int(q_lens[b]), 0), Q)
        pos = torch.arange(n, device=pool.k.device)
        pages = block_tables[b].long().to(pool.k.device)[pos // bs]
        if n - ql + 1 >= prefix_len > 0:
            head = pos < prefix_len
            pages[head] = prefix_pages.long().to(pool.k.device)[pos[head] // bs]
        if ((pages < 0) | (pages >= pool.k.shape[0])).any():
            raise InferenceError("a chain names a page outside of the pool")
        k = pool.k[pages, pos % bs].float().repeat_interleave(G, dim=1)
        v = pool.v[pages, pos % bs].float().repeat_interleave(G, dim=1)
        for t in range(ql):
            seen = n - ql + t + 1
            if seen > 0:
                s = torch.einsum("hd,thd->ht", q[b, t].float(), k[:seen]) * scale
                out[b, t] = torch.einsum("ht,thd->hd", torch.softmax(s, dim=-1), v[:seen]).to(torch.bfloat16)
    return out


def paged_attention_reference(q, pool: KvPagePool, block_tables, seq_lens, scale):
    """fp32 PyTorch restatement (oracle)."""
    B, H, HD = q.shape
    Hkv = pool.config.num_heads
    G = H // Hkv
    bs = pool.config.block_size
    out = torch.empty(B, H, HD, dtype=torch.bfloat16, device=q.device)
    for b in range(B):
        n = int(seq_lens[b])
        pages = block_tables[b, : (n + bs - 1) // bs].long().to(pool.k.device)
        k = pool.k[pages].reshape(-1, Hkv, HD)[:n].float()
        v = pool.v[pages].reshape(-1, Hkv, HD)[:n].float()
        k = k.repeat_interleave(G, dim=1)
        v = v.repeat_interleave(G, dim=1)
        s = torch.einsum("hd,thd->ht", q[b].float(), k) * scale
        p = torch.softmax(s, dim=-1)
        out[b] = torch.einsum("ht,thd->hd", p, v).to(torch.bfloat16)
    return out
