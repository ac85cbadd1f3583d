"""Paged key/value cache for decoding on the GPU.

A :class:`KvPagePool` owns two device tensors [num_pages, block_size, Hkv, HD]
(bf16) and a host free list; a page id names one page in both. The
:class:`BlockManager` maps sequence ids to page chains, grows them as tokens
are appended, and keeps the device block table (int32 [max_sequences,
max_pages_per_seq]) that the decode kernel reads. Appending the K/V of any
number of tokens of any sequences is one kernel launch.

Pages are reference-counted, so sequences may share them: a forked sequence
(:meth:`BlockManager.fork_sequence`) starts on its parent's pages, and
:meth:`BlockManager.reserve` gives a sequence its own copy of a shared page
before it writes there. :func:`copy_pages` copies pages in every layer's pool
in one launch (scirs_b200/csrc/page_copy.cu); :meth:`BlockManager.compact`
uses it to move the pages in use to the front of the pool.

Names and semantics follow the reference's inference module
(scirs2-neural/src/inference/kv_page.rs:27-340 KvPageConfig / KvPage /
KvPagePool, block_manager.rs:30-280 BlockManagerConfig / BlockManager /
SharedPrefixCache); there the pages are ndarray buffers on the host.
"""
from __future__ import annotations

import hashlib
from dataclasses import dataclass

import torch

from .. import _ext
from ..ops import kernels as K


class InferenceError(RuntimeError):
    pass


@dataclass
class KvPageConfig:
    block_size: int = 16
    num_heads: int = 8
    head_dim: int = 64
    dtype_bytes: int = 2

    @property
    def page_bytes(self) -> int:
        return 2 * self.block_size * self.num_heads * self.head_dim * self.dtype_bytes


class KvPagePool:
    def __init__(self, num_pages: int, config: KvPageConfig, device="cuda"):
        c = config
        self.config = c
        self.device = torch.device(device)
        shape = (num_pages, c.block_size, c.num_heads, c.head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._used: set[int] = set()
        self._shared: dict[int, int] = {}  # references of the pages that have more than one
        self._tick = 0
        self._last_use: dict[int, int] = {}

    def alloc_page(self) -> int:
        if not self._free:
            raise InferenceError("KV page pool exhausted")
        pid = self._free.pop()
        self._used.add(pid)
        self._touch(pid)
        return pid

    def retain_page(self, pid: int) -> None:
        """One more holder of the page; each holder gives it back by free_page."""
        if pid not in self._used:
            raise InferenceError(f"page {pid} is not allocated")
        self._shared[pid] = self._shared.get(pid, 1) + 1

    def ref_count(self, pid: int) -> int:
        return self._shared.get(pid, 1) if pid in self._used else 0

    def free_page(self, pid: int) -> None:
        """Give the page back; it is free again when its last holder has."""
        if pid not in self._used:
            raise InferenceError(f"page {pid} is not allocated")
        refs = self._shared.get(pid, 1)
        if refs > 1:
            self._shared[pid] = refs - 1
            if refs == 2:
                del self._shared[pid]
            return
        self._used.remove(pid)
        self._last_use.pop(pid, None)
        self._free.append(pid)

    def _move(self, moves: dict[int, int]) -> None:
        """What the pages `moves` (used -> free) hold, and their references and ages, change places."""
        taken = set(moves.values())
        self._free = [p for p in self._free if p not in taken] + list(moves)
        self._used = (self._used - moves.keys()) | taken
        for d in (self._shared, self._last_use):
            for old, new in moves.items():
                if old in d:
                    d[new] = d.pop(old)

    def _touch(self, pid: int):
        self._tick += 1
        self._last_use[pid] = self._tick

    def free_count(self) -> int:
        return len(self._free)

    def total_count(self) -> int:
        return self.k.shape[0]

    def memory_bytes(self) -> int:
        return self.total_count() * self.config.page_bytes

    def lru_candidates(self):
        """Allocated pages, least recently written first."""
        return [p for p, _ in sorted(self._last_use.items(), key=lambda kv: kv[1])]

    def write_kv(self, pid: int, slot: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write one token's K/V ([Hkv, HD]) into a page slot (host-driven
        path; the batched path is BlockManager.append)."""
        if pid not in self._used or not 0 <= slot < self.config.block_size:
            raise InferenceError("slot out of range")
        self.k[pid, slot].copy_(k)
        self.v[pid, slot].copy_(v)
        self._touch(pid)

    def read_kv(self, pid: int, slot: int):
        return self.k[pid, slot], self.v[pid, slot]


def copy_pages(pools, src, dst, counts=None) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in each of ``pools`` (a :class:`KvPagePool` or a
    list of alike ones, such as the layers'), keys and values, on the current stream: in one launch,
    as far as there are up to 128 pools and 1024 pages.

    ``src``, ``dst`` and ``counts`` are lists or int32 host tensors; ``counts[i]`` limits the copy
    to the first so many slots of a page (default: all of them), the others keep what they hold.
    A page may be copied to several others, but no page may be written twice, or be both read and
    written. The page ids are taken at the call: a captured graph replays the same copies. Pages
    whose slots are not a multiple of 16 bytes are refused on the GPU."""
    pools = [pools] if isinstance(pools, KvPagePool) else list(pools)
    if not pools:
        raise InferenceError("copy_pages needs at least one pool")

    src, dst, counts = (t if t is None or isinstance(t, torch.Tensor) else torch.tensor(list(t), dtype=torch.int32)
                        for t in (src, dst, counts))
    bufs = [b for p in pools for b in (p.k, p.v)]
    if bufs[0].is_cuda:
        K._count(_ext.kernels().page_copy(bufs, src, dst, counts))
        return
    for t in (src, dst, counts):
        if t is not None and (t.is_cuda or t.dtype != torch.int32 or t.shape != (src.numel(),)):
            raise InferenceError("page ids and counts are lists or 1-D int32 host tensors of one length")
    pages, bs = bufs[0].shape[:2]
    s, d = src.tolist(), dst.tolist()
    n = counts.tolist() if counts is not None else [bs] * len(s)
    if any(b.shape != bufs[0].shape or b.dtype != bufs[0].dtype or b.device != bufs[0].device for b in bufs):
        raise InferenceError("pools must be alike in device, shape and type")
    if any(not 0 <= x < pages for x in s + d) or any(not 0 <= x <= bs for x in n):
        raise InferenceError("page or slot count out of range")
    if len(set(d)) < len(d) or set(d) & set(s):
        raise InferenceError("a page is written twice, or both read and written")
    for b in bufs:
        for i, j, c in zip(s, d, n):
            b[j, :c] = b[i, :c]


@dataclass
class BlockManagerConfig:
    max_sequences: int = 64
    max_pages_per_seq: int = 128


class BlockManager:
    """Page chains of the active sequences. ``pools`` lists every pool that is indexed by the chains
    (the layers' pools; default: ``pool`` alone): pages are copied in all of them."""

    def __init__(self, pool: KvPagePool, config: BlockManagerConfig | None = None, pools=None):
        self.pool = pool
        self.pools = list(pools) if pools is not None else [pool]
        self.config = config or BlockManagerConfig()
        c = self.config
        self.block_tables = torch.zeros(c.max_sequences, c.max_pages_per_seq, dtype=torch.int32,
                                        device=pool.device)
        self._bt_host = torch.zeros(c.max_sequences, c.max_pages_per_seq, dtype=torch.int32)
        self.seq_lens = torch.zeros(c.max_sequences, dtype=torch.int32, device=pool.device)
        self._lens: dict[int, int] = {}
        self._pages: dict[int, list[int]] = {}
        self._row: dict[int, int] = {}
        self._free_rows = list(range(c.max_sequences - 1, -1, -1))
        self._dirty = False

    # ---------------------------------------------------------------- chains
    def allocate_sequence(self, seq_id: int) -> None:
        if seq_id in self._pages:
            raise InferenceError(f"sequence {seq_id} already exists")
        if not self._free_rows:
            raise InferenceError("too many active sequences")
        self._row[seq_id] = self._free_rows.pop()
        self._pages[seq_id] = []
        self._lens[seq_id] = 0
        try:
            self.extend_sequence(seq_id)
        except InferenceError:  # no page for it: leave no half-created sequence behind
            self._free_rows.append(self._row.pop(seq_id))
            del self._pages[seq_id], self._lens[seq_id]
            raise

    def extend_sequence(self, seq_id: int) -> int:
        pages = self._pages[seq_id]
        if len(pages) >= self.config.max_pages_per_seq:
            raise InferenceError("sequence exceeds max_pages_per_seq")
        pid = self.pool.alloc_page()
        self._bt_host[self._row[seq_id], len(pages)] = pid
        pages.append(pid)
        self._dirty = True
        return pid

    def fork_sequence(self, parent: int, child: int) -> None:
        """A new sequence with the parent's tokens, on the parent's pages: nothing is copied until
        one of the two writes into a page that they share (see reserve)."""
        if parent not in self._pages:
            raise InferenceError(f"sequence {parent} does not exist")
        if child in self._pages:
            raise InferenceError(f"sequence {child} already exists")
        if not self._free_rows:
            raise InferenceError("too many active sequences")
        n, bs = self._lens[parent], self.pool.config.block_size
        pages = self._pages[parent][: max(1, (n + bs - 1) // bs)]
        for pid in pages:
            self.pool.retain_page(pid)
        row = self._free_rows.pop()
        self._row[child], self._pages[child], self._lens[child] = row, list(pages), n
        self._bt_host[row, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self._dirty = True

    def truncate_sequence(self, seq_id: int, length: int) -> None:
        """Drop the tokens from position `length` on (rejected drafts); pages that hold none of the
        remaining ones are given back, all but the first."""
        if not 0 <= length <= self._lens[seq_id]:
            raise InferenceError(f"sequence {seq_id} has {self._lens[seq_id]} tokens, not {length}")
        bs, pages, row = self.pool.config.block_size, self._pages[seq_id], self._row[seq_id]
        while len(pages) > max(1, (length + bs - 1) // bs):
            self.pool.free_page(pages.pop())
            self._bt_host[row, len(pages)] = 0
        self._lens[seq_id] = length
        self._dirty = True

    def shared_prefix(self, seq_ids: list[int]) -> tuple[list[int], int]:
        """The leading pages that the chains of all these sequences have in common and are full in
        every one of them, and how many tokens they hold."""
        bs = self.pool.config.block_size
        if any(self._pages[s][0] != self._pages[seq_ids[0]][0] for s in seq_ids):  # (the usual case first)
            return [], 0
        common = min(self._lens[s] for s in seq_ids) // bs if seq_ids else 0
        first = self._pages[seq_ids[0]][:common] if common else []
        for s in seq_ids[1:]:
            other = self._pages[s]
            i = 0
            while i < len(first) and first[i] == other[i]:
                i += 1
            first = first[:i]
        return first, len(first) * bs

    def compact(self) -> dict[int, int]:
        """Move the chains' pages to the front of the pool, into the free pages there, and return
        {old page: new page}. Pages that something else holds too (retain_page, alloc_page, a
        SharedPrefixCache with the pool) stay."""
        pool = self.pool
        held: dict[int, int] = {}
        for pages in self._pages.values():
            for pid in pages:
                held[pid] = held.get(pid, 0) + 1
        movable = sorted((p for p, n in held.items() if pool.ref_count(p) == n), reverse=True)
        moves: dict[int, int] = {}
        for old, new in zip(movable, sorted(pool._free)):
            if new >= old:
                break
            moves[old] = new
        if not moves:
            return moves
        copy_pages(self.pools, list(moves), list(moves.values()))
        pool._move(moves)
        for seq, pages in self._pages.items():
            pages[:] = [moves.get(p, p) for p in pages]
            self._bt_host[self._row[seq], : len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self._dirty = True
        return moves

    def free_sequence(self, seq_id: int) -> None:
        for pid in self._pages.pop(seq_id):
            self.pool.free_page(pid)
        row = self._row.pop(seq_id)
        self._lens.pop(seq_id)
        self._bt_host[row].zero_()
        self._free_rows.append(row)
        self._dirty = True

    def sequence_page_chain(self, seq_id: int) -> list[int]:
        return list(self._pages[seq_id])

    def seq_len(self, seq_id: int) -> int:
        return self._lens[seq_id]

    def row_of(self, seq_id: int) -> int:
        return self._row[seq_id]

    def active_sequences(self) -> int:
        return len(self._pages)

    def sync(self):
        """Upload the block table and lengths if they changed."""
        if self._dirty:
            self.block_tables.copy_(self._bt_host, non_blocking=True)
            lens = torch.zeros(self.config.max_sequences, dtype=torch.int32)
            for s, n in self._lens.items():
                lens[self._row[s]] = n
            self.seq_lens.copy_(lens, non_blocking=True)
            self._dirty = False

    # ---------------------------------------------------------------- writes
    def reserve(self, seq_ids: list[int], counts: list[int]):
        """Grow chains for `counts` new tokens per sequence; returns the
        (row, position) of every new token in order. A page that other holders share and that would
        be written is copied first (its slots before the new tokens), and the copy takes its place."""
        rows, pos = [], []
        bs = self.pool.config.block_size
        # all or nothing: check the whole batch's page needs before changing any sequence
        need, lens = {}, dict(self._lens)
        for s, n in zip(seq_ids, counts):
            lens[s] += n
            need[s] = max(0, (lens[s] + bs - 1) // bs - len(self._pages[s]))
        own = self._pages_to_own(lens)
        if any(len(self._pages[s]) + k > self.config.max_pages_per_seq for s, k in need.items()):
            raise InferenceError("sequence exceeds max_pages_per_seq")
        if sum(need.values()) + len(own) > self.pool.free_count():
            raise InferenceError("KV page pool exhausted")
        self._own_pages(own)
        for s, n in zip(seq_ids, counts):
            start = self._lens[s]
            while (start + n + bs - 1) // bs > len(self._pages[s]):
                self.extend_sequence(s)
            rows += [self._row[s]] * n
            pos += list(range(start, start + n))
            self._lens[s] = start + n
            self._dirty = True
        return rows, pos

    def _pages_to_own(self, lens: dict[int, int]) -> list[tuple[int, int]]:
        """(sequence, index in its chain) of the shared pages that sequences growing to `lens` tokens
        write; the last holder of a page keeps it."""
        bs, out = self.pool.config.block_size, []
        if not self.pool._shared:
            return out
        refs: dict[int, int] = {}
        for s, end in lens.items():
            pages = self._pages[s]
            if end == self._lens[s]:
                continue
            for i in range(self._lens[s] // bs, min(len(pages), (end + bs - 1) // bs)):
                r = refs.get(pages[i], self.pool.ref_count(pages[i]))
                if r > 1:
                    refs[pages[i]] = r - 1
                    out.append((s, i))
        return out

    def _own_pages(self, own: list[tuple[int, int]]) -> None:
        if not own:
            return
        bs, src, dst, counts = self.pool.config.block_size, [], [], []
        for s, i in own:
            src.append(self._pages[s][i])
            dst.append(self.pool.alloc_page())
            counts.append(min(max(self._lens[s] - i * bs, 0), bs))
        try:
            copy_pages(self.pools, src, dst, counts)
        except Exception:  # refused: no page changes hands
            for pid in dst:
                self.pool.free_page(pid)
            raise
        for (s, i), old, new in zip(own, src, dst):
            self.pool.free_page(old)
            self._pages[s][i] = new
            self._bt_host[self._row[s], i] = new
        self._dirty = True

    def append(self, seq_ids: list[int], counts: list[int], k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Write the K/V ([n, Hkv, HD], n = sum(counts), sequences in order)
        of new tokens into their pages (one kernel launch)."""
        rows, pos = self.reserve(seq_ids, counts)
        self.sync()
        dev = self.pool.device
        r = torch.tensor(rows, dtype=torch.int32).to(dev, non_blocking=True)
        p = torch.tensor(pos, dtype=torch.int32).to(dev, non_blocking=True)
        if k_new.is_cuda:
            _ext.kernels().paged_kv_append(k_new.contiguous(), v_new.contiguous(), self.pool.k, self.pool.v,
                                           self.block_tables, r, p)
        else:
            bs = self.pool.config.block_size
            for i, (row, ps) in enumerate(zip(rows, pos)):
                pid = int(self._bt_host[row, ps // bs])
                self.pool.k[pid, ps % bs] = k_new[i]
                self.pool.v[pid, ps % bs] = v_new[i]

    def write_token_kv(self, seq_id: int, k: torch.Tensor, v: torch.Tensor) -> None:
        self.append([seq_id], [1], k.reshape(1, *k.shape), v.reshape(1, *v.shape))


class SharedPrefixCache:
    """Maps a prompt-prefix hash to the page chain that holds its K/V, so
    sequences with a common prompt can reuse the pages.

    With the chains' `pool` the cache holds every page that it lists (insert
    retains it, evict gives it back): a listed page is not reused when its
    sequences end, not written by the ones that go on, and not moved by
    BlockManager.compact. Without one it keeps page ids alone, which those
    calls make stale."""

    def __init__(self, pool: KvPagePool | None = None):
        self._pool = pool
        self._map: dict[int, list[int]] = {}

    def lookup(self, prefix_hash: int):
        return self._map.get(prefix_hash)

    def insert(self, prefix_hash: int, pages: list[int]) -> None:
        pages = list(pages)
        if self._pool is not None:
            for pid in pages:
                if self._pool.ref_count(pid) == 0:
                    raise InferenceError(f"page {pid} is not allocated")
            for pid in pages:
                self._pool.retain_page(pid)
        self.evict(prefix_hash)
        self._map[prefix_hash] = pages

    def evict(self, prefix_hash: int):
        pages = self._map.pop(prefix_hash, None)
        if self._pool is not None:
            for pid in pages or ():
                self._pool.free_page(pid)
        return pages

    def __len__(self):
        return len(self._map)

    def is_empty(self) -> bool:
        return not self._map

    @staticmethod
    def compute_prefix_hash(tokens) -> int:
        b = b"".join(int(t).to_bytes(4, "little") for t in tokens)
        return int.from_bytes(hashlib.blake2b(b, digest_size=8).digest(), "little")
