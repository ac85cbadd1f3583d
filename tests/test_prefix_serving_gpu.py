"""Shared-prefix paged attention, page copies and draft verification on the GPU against plain implementations in 64
bits, at the sizes and masks where they can go wrong, and the three together in a serving loop."""
import math

import pytest
import torch

from scirs_b200 import _ext
from scirs_b200.inference import (BlockManager, BlockManagerConfig, GPTGenerator, KvPageConfig, KvPagePool,
                                  PagedAttentionConfig, PagedAttentionForward, copy_pages, verify_drafts)
from scirs_b200.models.gpt import GPTConfig, GPTModel

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


# ------------------------------------------------------------------------------------------------ attention
class Case:
    """A cache with a prefix of L tokens and a tail of each sequence, pages in random order."""

    def __init__(self, lens, Q, Hkv, G, HD, bs, L, qlens=None, seed=0, spare=2, scale=1.5):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Q, self.Hkv, self.G, self.HD, self.bs, self.L = len(lens), Q, Hkv, G, HD, bs, L
        per = max(1, -(-max(lens + [L]) // bs))
        front = -(-L // bs)
        n = front + self.B * per + spare
        ids = torch.randperm(n, generator=g).to(torch.int32)
        k, v = (torch.randn(n, bs, Hkv, HD, generator=g).to(torch.bfloat16) for _ in range(2))
        self.prefix_pages = ids[:front].clone()
        self.tables = ids[front:front + self.B * per].view(self.B, per).clone()
        # the sequences' own pages hold the prefix's tokens too, as far as they are pages of their own
        at = torch.arange(L)
        for b in range(self.B):
            for x in (k, v):
                x[self.tables[b].long()[at // bs], at % bs] = x[self.prefix_pages.long()[at // bs], at % bs]
        # slots that no sequence holds are not to be read
        used = torch.zeros(n, bs, dtype=torch.bool)
        used[self.prefix_pages.long()[at // bs], at % bs] = True
        for b, m in enumerate(lens):
            pos = torch.arange(m)
            used[self.tables[b].long()[pos // bs], pos % bs] = True
        k[~used] = float("nan")
        v[~used] = float("nan")
        self.q = (torch.randn(self.B, Q, Hkv * G, HD, generator=g) * scale).to(torch.bfloat16)
        self.k, self.v = k, v
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.qlens = None if qlens is None else torch.tensor(qlens, dtype=torch.int32)
        self.att = PagedAttentionForward(PagedAttentionConfig(Hkv * G, HD))
        self.scale = HD ** -0.5

    def pool(self):
        p = KvPagePool(0, KvPageConfig(block_size=self.bs, num_heads=self.Hkv, head_dim=self.HD), DEV)
        p.k, p.v = self.k.to(DEV), self.v.to(DEV)
        return p

    def run(self, q=None, pool=None, tables=None):
        out = self.att.forward_shared_prefix(
            self.q.to(DEV) if q is None else q, pool or self.pool(), self.tables.to(DEV) if tables is None else tables,
            self.lens.to(DEV), self.prefix_pages.to(DEV), self.L, None if self.qlens is None else self.qlens.to(DEV))
        torch.cuda.synchronize()
        return out

    def exact(self):
        """(output, sum of p |v|) in 64 bits, key by key of each query."""
        o = torch.zeros(self.B, self.Q, self.Hkv * self.G, self.HD, dtype=torch.float64)
        a = torch.zeros_like(o)
        for b in range(self.B):
            m = min(int(self.lens[b]), self.tables.shape[1] * self.bs)
            ql = self.Q if self.qlens is None else int(self.qlens[b])
            pos = torch.arange(m)
            page = self.tables[b].long()[pos // self.bs]
            k, v = self.k[page, pos % self.bs].double(), self.v[page, pos % self.bs].double()
            for t in range(ql):
                seen = m - ql + t + 1
                if seen <= 0:
                    continue
                for h in range(self.Hkv * self.G):
                    s = k[:seen, h // self.G] @ self.q[b, t, h].double() * self.scale
                    p = torch.softmax(s, 0)
                    o[b, t, h] = p @ v[:seen, h // self.G]
                    a[b, t, h] = p @ v[:seen, h // self.G].abs()
        return o, a

    def check(self, out):
        """|error| <= half a bf16 step of the output + (half a bf16 step of each probability, and 2^-11 for
        the fp32 scores, exponentials and sums) of sum p |v|. A score is off by at most HD 2^-24 sum|q k|
        scale <= 128 * 2^-24 * 40 = 2^-11.7 (sum |q k| scale stays below 40 at q of 1.5 and k of 1 standard
        deviation and HD <= 128), the exponential by 2^-22, and the sums by less than 2^-18."""
        _ext.check_status(0)
        o, a = self.exact()
        assert out.dtype == torch.bfloat16 and out.shape == (o.shape if self.q.dim() == 4 else o[:, 0].shape)
        err = (out.cpu().double().view_as(o) - o).abs()
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * a + 1e-30
        assert torch.isfinite(out).all()
        assert (err <= tol).all(), float((err / tol).max())


CASES = [
    # lens, Q, Hkv, G, HD, bs, L, qlens
    pytest.param([1], 1, 1, 1, 64, 16, 0, None, id="one_token"),
    pytest.param([1, 2, 5], 1, 2, 4, 128, 16, 1, None, id="prefix_of_one"),
    pytest.param([16, 17, 40, 0], 1, 2, 3, 64, 16, 16, None, id="tails_of_zero_and_padding"),
    pytest.param([70, 64, 65, 200], 1, 3, 5, 128, 16, 64, None, id="groups_of_five"),
    pytest.param([37, 40, 90], 4, 2, 2, 64, 16, 35, [1, 4, 3], id="ragged_queries_prefix_inside_page"),
    pytest.param([600, 601, 1000], 1, 1, 8, 128, 32, 513, None, id="many_splits"),
    pytest.param([300] * 9, 1, 1, 16, 64, 24, 290, None, id="rows_over_one_tile"),
    pytest.param([150, 131, 140, 0, 135], 8, 2, 7, 128, 5, 128, [8, 2, 0, 3, 7], id="pages_of_five_no_queries"),
    pytest.param([20, 3, 50, 1], 4, 2, 2, 64, 8, 30, [4, 3, 4, 1], id="shorter_than_the_prefix"),
    pytest.param([5, 40], 6, 1, 2, 32, 16, 0, None, id="no_prefix_more_queries_than_tokens"),
    pytest.param([2000, 1999, 2100], 2, 2, 1, 8, 16, 1990, [2, 2, 1], id="head_dim_8"),
    pytest.param([90, 80], 1, 2, 2, 40, 1, 77, None, id="head_dim_40_pages_of_one"),
    pytest.param([90, 130, 100], 3, 2, 2, 80, 64, 64, [1, 2, 3], id="head_dim_80"),
    pytest.param([90, 130, 100], 1, 4, 1, 96, 128, 88, None, id="head_dim_96_page_of_128"),
    pytest.param([257 + 3 * i for i in range(40)], 1, 2, 4, 128, 16, 256, None, id="forty_sequences"),
    pytest.param([400 + i for i in range(70)], 2, 1, 4, 64, 16, 397, [1 + i % 2 for i in range(70)], id="seventy_by_two"),
    pytest.param([1500 + 7 * i for i in range(33)], 1, 2, 8, 128, 16, 1493, None, id="three_row_tiles"),
    # 33 to 128 rows a cached head, and more, against prefixes of two blocks and more
    pytest.param([260, 270, 0, 300, 259], 1, 2, 8, 128, 16, 259, None, id="forty_rows"),
    pytest.param([2100 + i for i in range(25)], 4, 1, 1, 64, 24, 2100 - 4, [1 + i % 4 for i in range(25)], id="hundred_rows"),
    pytest.param([700, 30, 701, 0, 699] * 5, 2, 3, 5, 96, 32, 690, [2, 1, 0, 2, 1] * 5, id="rows_that_take_no_part"),
    pytest.param([1025] * 20, 1, 1, 2, 40, 5, 1024, None, id="tc_head_dim_40_pages_of_five"),
    pytest.param([257 + i for i in range(64)], 1, 1, 2, 128, 16, 257, None, id="tails_of_none_128_rows"),
    pytest.param([520 + i for i in range(129)], 1, 1, 1, 64, 16, 512, None, id="129_rows"),
    pytest.param([4000 + i for i in range(6)], 1, 16, 7, 64, 128, 3999, None, id="sixteen_heads"),
    pytest.param([5000 + 3 * i for i in range(40)], 1, 1, 16, 128, 16, 4990, None, id="640_rows_long"),
    pytest.param([600, 520, 0, 513, 700, 640], 1, 2, 8, 128, 16, 513, None, id="48_rows_prefix_inside_page"),
    pytest.param([33000], 1, 1, 1, 64, 128, 32990, None, id="one_row_long"),
    pytest.param([33000, 40, 32800], 2, 1, 2, 128, 8, 32780, [2, 1, 1], id="twelve_rows_long"),
    pytest.param([600 + i for i in range(9)], 1, 1, 2, 72, 16, 597, None, id="tc_head_dim_72"),
    # more short tails than two rounds of CTAs
    pytest.param([291 + i % 20 for i in range(130)], 1, 8, 1, 64, 16, 290, None, id="1040_short_tails"),
    pytest.param([1 + i % 30 for i in range(100)], 3, 8, 2, 128, 5, 0, [1 + i % 3 for i in range(100)], id="800_tails_no_prefix"),
    pytest.param([0 if i % 7 == 0 else 20 + i % 90 for i in range(130)], 2, 8, 1, 128, 8, 17, [i % 3 for i in range(130)], id="short_tails_shorter_than_prefix"),
]


@pytest.mark.parametrize("lens,Q,Hkv,G,HD,bs,L,qlens", CASES)
def test_attention_matches_the_definition(lens, Q, Hkv, G, HD, bs, L, qlens):
    c = Case(lens, Q, Hkv, G, HD, bs, L, qlens, seed=len(lens) + L)
    if Q == 1:
        c.q = c.q[:, 0]
        out = c.run()
        c.q = c.q[:, None]
        assert out.dim() == 3
        out = out[:, None]
    else:
        out = c.run()
    c.check(out)


def test_attention_agrees_with_the_decode_kernel():
    c = Case([300, 260, 257], 1, 2, 4, 64, 16, 256)
    pool = c.pool()
    a = c.run(pool=pool)[:, 0].float()
    b = c.att.forward_batch(c.q[:, 0].to(DEV), pool, c.tables.to(DEV), c.lens.to(DEV)).float()
    # each is within half a step of its value and of its probabilities
    assert (a - b).abs().max() <= 2 * (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -11) * c.exact()[1].max()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), -3.3895e38])
@pytest.mark.parametrize("L", [0, 90, 600])
def test_masked_drafts_do_not_reach_earlier_queries(value, L):
    """The last drafted token's keys and values are not numbers: the queries before it do not see them."""
    n = max(100, L + 10)
    c = Case([n, n - 3] + [n - 2] * 3, 4, 1, 2, 64, 16, L, seed=3)
    page = c.tables[0].long()[(n - 1) // 16]
    c.k[page, (n - 1) % 16], c.v[page, (n - 1) % 16] = value, value
    out = c.run()
    seen = torch.isfinite(out).all(-1).cpu()
    assert seen[0, :3].all() and seen[1:].all()
    c.k[page, (n - 1) % 16], c.v[page, (n - 1) % 16] = 0.0, 0.0
    o, a = c.exact()
    err = (out.cpu().double() - o).abs()[:, :3]
    assert (err <= (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * a)[:, :3]).all()
    if value != value:
        assert torch.isnan(out[0, 3]).all()


def test_large_scores_and_equal_scores():
    c = Case([200, 130], 1, 1, 4, 64, 16, 128, scale=0.0)  # every key weighs the same
    c.check(c.run())
    # one key far above the others, first in the prefix and then in the tail
    for at in (5, 190):
        c = Case([200, 195], 1, 1, 2, 64, 16, 128)
        c.q[:] = 4.0
        for b in range(2):
            c.k[c.tables[b].long()[at // 16], at % 16] = 8.0
        if at < 128:
            c.k[c.prefix_pages.long()[at // 16], at % 16] = 8.0
        # 64 * 4 * 8 / 8 = 256 against scores of at most 4 * 64 * 5 / 8 = 160: the others underflow
        out = c.run().cpu().float()
        want = torch.stack([c.v[c.tables[b].long()[at // 16], at % 16, 0] for b in range(2)]).float()
        assert torch.equal(out[:, 0], want[:, None].expand(2, 2, 64))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows", [4, 80, 300])
def test_prefix_scores_that_are_no_numbers(value, rows):
    """A key of the prefix that is not a number spoils every row that sees it, wherever in a block it lies."""
    for L, at in [(264, 0), (264, 130), (264, 263), (700, 0), (700, 3), (700, 77), (700, 130), (700, 500), (700, 699)]:
        c = Case([L + 6] * rows, 1, 1, 1, 64, 16, L)
        c.q = c.q.abs() + 0.1
        c.k[c.prefix_pages.long()[at // 16], at % 16] = value
        assert torch.isnan(c.run()).all()
    c = Case([265] * 4, 1, 1, 1, 64, 16, 264)  # the only key of a tail
    for b in range(4):
        c.k[c.tables[b].long()[264 // 16], 264 % 16] = float("nan")
    assert torch.isnan(c.run()).all()


@pytest.mark.parametrize("L,copies", [(256, 1), (640, 3)])
def test_attention_strides_streams_and_graph(L, copies):
    c = Case([L + 44, L + 34, L + 54] * copies, 2, 2, 2, 64, 16, L, [1, 2, 2] * copies, seed=4)
    B = 3 * copies
    pool = c.pool()
    want = c.run(pool=pool)
    c.check(want)
    # q as a slice of a fused projection's output; an odd offset; tables of a wider matrix
    H = c.Hkv * c.G
    fused = torch.randn(B, 2, 3, H, 64, device=DEV).to(torch.bfloat16)
    fused[:, :, 1] = c.q.to(DEV)
    assert torch.equal(c.run(fused[:, :, 1], pool), want)
    odd = torch.empty(c.q.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view_as(c.q)
    odd.copy_(c.q)
    assert torch.equal(c.run(odd, pool), want)
    wide = torch.full((B, c.tables.shape[1] + 9), 12345, dtype=torch.int32, device=DEV)
    wide[:, : c.tables.shape[1]] = c.tables.to(DEV)
    assert torch.equal(c.run(pool=pool, tables=wide[:, : c.tables.shape[1]]), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(c.run(pool=pool), want)
    # captured twice, replayed on two streams at once with other lengths than at the capture
    args = [t.to(DEV) for t in (c.q, c.tables, c.lens, c.prefix_pages, c.qlens)]
    args[2].fill_(L + 4)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(c.att.forward_shared_prefix(args[0], pool, args[1], args[2], args[3], c.L, args[4]))
        graphs.append(gr)
    args[2].copy_(c.lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_attention_wide_tables_and_empty_batches():
    c = Case([40, 33], 1, 1, 2, 64, 16, 32)
    want = c.run()
    wide = torch.zeros(2, 4096, dtype=torch.int32)
    wide[:, : c.tables.shape[1]] = c.tables
    got = c.run(tables=wide.to(DEV))
    c.tables = wide
    c.check(got)
    assert (got.float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.abs().max()
    empty = c.att.forward_shared_prefix(c.q[:0].to(DEV), c.pool(), wide[:0].to(DEV), c.lens[:0].to(DEV),
                                        c.prefix_pages.to(DEV), 32)
    assert empty.shape == (0, 1, 2, 64)


def test_attention_bad_pages_and_lengths_are_reported():
    c = Case([100, 90, 95], 1, 2, 2, 64, 16, 64)
    good = c.run()
    _ext.check_status(0)
    keep = c.tables.clone()
    c.tables[1, 5] = 10 ** 6  # a page of the second sequence's tail
    out = c.run()
    with pytest.raises(RuntimeError, match="bounds"):
        _ext.check_status(0)
    assert torch.equal(out[[0, 2]], good[[0, 2]]) and torch.isfinite(out).all()
    c.tables = keep
    c.prefix_pages[2] = -1
    out = c.run()
    with pytest.raises(RuntimeError, match="bounds"):
        _ext.check_status(0)
    assert torch.isfinite(out).all()
    c = Case([100, 90, 95], 1, 2, 2, 64, 16, 64)
    c.lens[1] = 5000  # longer than its chain: the slots that the chain has are read
    c.k[:], c.v[:] = torch.nan_to_num(c.k), torch.nan_to_num(c.v)
    out = c.run()
    with pytest.raises(RuntimeError, match="bounds"):
        _ext.check_status(0)
    c.check(out)


@pytest.mark.parametrize("bs", [5, 16])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_bad_prefix_pages_are_reported_by_the_long_prefix_path(bs, bad):
    c = Case([650 + i for i in range(20)], 1, 2, 2, 64, bs, 640)
    c.k, c.v = torch.nan_to_num(c.k), torch.nan_to_num(c.v)
    c.check(c.run())
    c.prefix_pages[7] = bad
    out = c.run()
    with pytest.raises(RuntimeError, match="bounds"):
        _ext.check_status(0)
    assert torch.isfinite(out).all()


def test_attention_refuses():
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        c = Case([40, 33], 1, 2, 2, 64, 16, 32)
        c.att.config.scale = scale
        with pytest.raises(RuntimeError, match="scale"):
            c.run()
    c = Case([40, 33], 1, 2, 2, 64, 16, 32)
    pool = c.pool()
    q, t, n, p = c.q.to(DEV), c.tables.to(DEV), c.lens.to(DEV), c.prefix_pages.to(DEV)
    f = c.att.forward_shared_prefix
    for bad in [(q, pool, t.long(), n, p, 32), (q, pool, t, n.long(), p, 32), (q, pool, t[:1], n, p, 32),
                (q, pool, t, n[:1], p, 32), (q, pool, t, n, p.long(), 32), (q, pool, t.cpu(), n, p, 32),
                (q, pool, t, n, p, 33), (q, pool, t, n, p, 32, torch.ones(3, dtype=torch.int32, device=DEV)),
                (q, pool, t, n, p, 32, torch.ones(2, device=DEV))]:
        with pytest.raises((RuntimeError, ValueError)):
            f(*bad)
    for hd in (12, 136):
        c = Case([10], 1, 1, 1, hd, 4, 4)
        with pytest.raises(RuntimeError, match="head_dim"):
            c.run()


# ------------------------------------------------------------------------------------------------ page copies
@pytest.mark.parametrize("layers,pages,bs,heads,hd,moves,partial", [
    (1, 4, 16, 1, 8, 1, False), (3, 40, 5, 3, 40, 7, True), (12, 64, 16, 12, 64, 8, True), (2, 9, 1, 2, 128, 4, False),
    (1, 5000, 2, 1, 32, 2300, True), (140, 6, 3, 2, 16, 3, True), (4, 30, 64, 8, 128, 15, False)])
def test_copy_pages(layers, pages, bs, heads, hd, moves, partial):
    g = torch.Generator().manual_seed(pages)
    pools = [KvPagePool(pages, KvPageConfig(block_size=bs, num_heads=heads, head_dim=hd), DEV) for _ in range(layers)]
    for p in pools:
        p.k.normal_()
        p.v.normal_()
    before = [(p.k.clone(), p.v.clone()) for p in pools]
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    src, dst = perm[:moves].clone(), perm[moves:2 * moves].clone()
    if moves > 2:
        src[1] = src[0]  # one page to two places
    counts = torch.randint(0, bs + 1, (moves,), generator=g).to(torch.int32) if partial else None
    copy_pages(pools, src, dst, counts)
    full = torch.arange(bs)[None, :] < (counts[:, None] if partial else bs)
    for p, (k, v) in zip(pools, before):
        for new, old in ((p.k, k), (p.v, v)):
            want = old.clone()
            d, s = dst.long().to(DEV), src.long().to(DEV)
            want[d] = torch.where(full.to(DEV)[:, :, None, None], old[s], old[d])
            assert torch.equal(new, want)


def test_copy_pages_refuses_and_captures():
    pools = [KvPagePool(8, KvPageConfig(block_size=4, num_heads=2, head_dim=8), DEV) for _ in range(2)]
    for p in pools:
        p.k.normal_()
        p.v.normal_()
    state = [(p.k.clone(), p.v.clone()) for p in pools]
    for src, dst, counts in [([0], [8], None), ([-1], [1], None), ([0, 1], [2, 2], None), ([0, 1], [1, 2], None),
                             ([0], [1], [5]), ([0], [1], [-1])]:
        with pytest.raises(RuntimeError):
            copy_pages(pools, src, dst, counts)
    with pytest.raises(RuntimeError):  # 10 bytes a slot
        copy_pages(KvPagePool(4, KvPageConfig(block_size=4, num_heads=1, head_dim=5), DEV), [0], [1])
    with pytest.raises(RuntimeError):
        copy_pages([pools[0], KvPagePool(7, pools[0].config, DEV)], [0], [1])
    copy_pages(pools, [], [])
    assert all(torch.equal(p.k, k) and torch.equal(p.v, v) for p, (k, v) in zip(pools, state))
    gr = torch.cuda.CUDAGraph()
    src, dst = [0, 1], [5, 6]
    with torch.cuda.graph(gr):
        copy_pages(pools, src, dst)
    src[0] = 3  # the graph keeps what it was given
    for p in pools:
        p.k[5:7], p.v[5:7] = 0, 0
    gr.replay()
    torch.cuda.synchronize()
    for p, (k, v) in zip(pools, state):
        assert torch.equal(p.k[5:7], k[:2]) and torch.equal(p.v[5:7], v[:2]) and torch.equal(p.k[:5], k[:5])


# ------------------------------------------------------------------------------------------------ verification
def _verify_exact(p, q, x, u, lens, threshold):
    """From the definition, in 64 bits on the host."""
    B, n = x.shape
    V = p.shape[2]
    kept, tokens = [], torch.full((B, n + 1), -1, dtype=torch.int64)
    for b in range(B):
        i = 0
        m = n if lens is None else min(max(int(lens[b]), 0), n)
        while i < m and 0 <= int(x[b, i]) < V:
            px = float(p[b, i, x[b, i]])
            qx = 1.0 if q is None else float(q[b, i, x[b, i]])
            ui = float(u[b, i])
            if not ((ui * qx < px or ui < threshold) if qx > 0 else px > 0):
                break
            tokens[b, i] = x[b, i]
            i += 1
        kept.append(i)
        w = p[b, i].double()
        rest = w.clone()
        if i < m:
            if q is not None:
                rest = w - q[b, i].double()
            elif 0 <= int(x[b, i]) < V:
                rest[x[b, i]] -= 1.0
        for y in (rest, w):
            y = torch.where((y > 0) & torch.isfinite(y), y, torch.zeros_like(y))
            if float(y.sum()) > 0:
                c = torch.cumsum(y, 0)
                past = torch.nonzero((c > float(u[b, n]) * c[-1]) & (y > 0))
                tokens[b, i] = int(past[0] if len(past) else torch.nonzero(y > 0)[-1])
                break
    return torch.tensor(kept, dtype=torch.int32), tokens


@pytest.mark.parametrize("B,n,V,dtype,ragged,with_draft,pad,threshold", [
    (1, 4, 50257, torch.float32, False, True, 0, 0.0), (7, 1, 1, torch.float32, False, True, 0, 0.0),
    (33, 5, 50257, torch.bfloat16, True, True, 47, 0.0), (16, 3, 1000, torch.float16, True, False, 3, 0.1),
    (64, 40, 63, torch.float32, True, True, 1, 0.0), (5, 0, 777, torch.float32, False, False, 0, 0.0),
    (9, 8, 131072, torch.float32, False, True, 0, 0.3), (300, 2, 65, torch.bfloat16, False, True, 0, 0.0),
    (256, 3, 32768, torch.float32, True, True, 0, 0.0), (200, 4, 9001, torch.float16, True, False, 2, 0.2)])
def test_verify_matches_the_definition(B, n, V, dtype, ragged, with_draft, pad, threshold):
    g = torch.Generator().manual_seed(V + n)
    lp = torch.randn(B, n + 1, V, generator=g) * 2
    lq = lp[:, :n] + torch.randn(B, n, V, generator=g) * 0.5
    p, q = torch.softmax(lp, -1).to(dtype), torch.softmax(lq, -1).to(dtype)
    x = torch.zeros(B, 0, dtype=torch.int64)
    if n:
        x = torch.multinomial(q.float().view(B * n, V), 1, generator=g).view(B, n)
    u = torch.rand(B, n + 1, generator=g)
    lens = torch.randint(0, n + 1, (B,), generator=g).to(torch.int32) if ragged else None
    pd = torch.full((B, n + 1, V + pad), float("nan"), dtype=dtype, device=DEV)[..., :V]
    pd.copy_(p)
    got = verify_drafts(pd, q.to(DEV) if with_draft else None, x.to(DEV), u.to(DEV),
                        None if lens is None else lens.to(DEV), threshold)
    kept, tokens = _verify_exact(p, q if with_draft else None, x, u, lens, threshold)
    assert torch.equal(got.accepted.cpu(), kept)
    assert torch.equal(got.tokens.cpu(), tokens)


def test_verify_edges():
    V = 3000
    p = torch.zeros(8, 2, V)
    q = torch.zeros(8, 1, V)
    x = torch.zeros(8, 1, dtype=torch.int64)
    u = torch.full((8, 2), 0.5)
    p[0, 0, 5] = q[0, 0, 5] = 1.0  # equal: p = q = 0 at the draft, refused; the row itself is drawn from
    p[1, 0, V - 1] = 1.0  # the last entry
    p[2], q[2] = float("nan"), float("nan")
    p[3, 0, 7] = float("inf")
    p[3, 0, 9] = 1e-30  # the infinity counts as nothing
    p[4, 0, 0], q[4, 0, 0], u[4, 0] = 0.25, 0.5, 0.5  # u q = p: refused
    p[4, 0, 11] = 1.0
    p[5, 0, 0], q[5, 0, 0], u[5, 0] = 0.25, 0.5, 0.49999997
    p[5, 1, 2998], p[5, 1, 2999], u[5, 1] = 0.5, 0.5, 0.5  # the first half ends exactly at the target
    x[6], p[6, 0, 3] = V, 1.0
    x[7], p[7, 0, 4] = -1, 1.0
    got = verify_drafts(p.to(DEV), q.to(DEV), x.to(DEV), u.to(DEV))
    assert got.accepted.tolist() == [0, 0, 0, 0, 0, 1, 0, 0]
    assert got.tokens.tolist() == [[5, -1], [V - 1, -1], [-1, -1], [9, -1], [11, -1], [0, 2999], [3, -1], [4, -1]]
    # not below one: refused (u q > p), and the last entry with weight is taken
    u = torch.full((8, 2), 1.0)
    got = verify_drafts(p.to(DEV), q.to(DEV), x.to(DEV), u.to(DEV))
    assert got.accepted.tolist() == [0] * 8
    assert got.tokens.tolist()[:5] == [[5, -1], [V - 1, -1], [-1, -1], [9, -1], [11, -1]]


def test_verify_strides_graph_and_refusals():
    B, n, V = 4, 3, 129
    g = torch.Generator().manual_seed(0)
    p = torch.softmax(torch.randn(B, n + 1, V, generator=g), -1)
    q = torch.softmax(torch.randn(B, n, V, generator=g), -1)
    x, u = torch.randint(0, V, (B, n), generator=g), torch.rand(B, n + 1, generator=g)
    kept, tokens = _verify_exact(p, q, x, u, None, 0.0)
    pd, qd, xd, ud = (t.to(DEV) for t in (p, q, x, u))
    for pv, qv in [(pd, qd), (pd.transpose(0, 1).contiguous().transpose(0, 1), qd),
                   (pd.transpose(1, 2).contiguous().transpose(1, 2), qd.transpose(1, 2).contiguous().transpose(1, 2))]:
        got = verify_drafts(pv, qv, xd, ud)
        assert torch.equal(got.accepted.cpu(), kept) and torch.equal(got.tokens.cpu(), tokens)
    gr = torch.cuda.CUDAGraph()
    u2 = torch.zeros_like(ud)
    with torch.cuda.graph(gr):
        got = verify_drafts(pd, qd, xd, u2)
    u2.copy_(ud)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.accepted.cpu(), kept) and torch.equal(got.tokens.cpu(), tokens)
    for bad in [(pd.double(), None, xd, ud), (pd, qd.half(), xd, ud), (pd, qd.cpu(), xd, ud), (pd, qd, xd.cpu(), ud),
                (pd, qd, xd, ud.cpu()), (pd, qd, xd, ud[:, :n])]:
        with pytest.raises((RuntimeError, ValueError)):
            verify_drafts(*bad)
    assert verify_drafts(pd[:0], qd[:0], xd[:0], ud[:0]).tokens.shape == (0, n + 1)


# ------------------------------------------------------------------------------------------------ together
def test_forked_sequences_over_shared_pages():
    """Fork, write, attend, drop, compact, attend again."""
    g = torch.Generator().manual_seed(2)
    Hkv, G, hd, bs, layers = 2, 2, 64, 16, 3
    pools = [KvPagePool(64, KvPageConfig(block_size=bs, num_heads=Hkv, head_dim=hd), DEV) for _ in range(layers)]
    bm = BlockManager(pools[0], BlockManagerConfig(8, 16), pools)
    want = {}

    def write(seqs, counts):
        rows, pos = bm.reserve(seqs, counts)
        bm.sync()
        kv = torch.randn(layers, 2, len(rows), Hkv, hd, generator=g).to(torch.bfloat16)
        r, p = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in (rows, pos))
        for layer, pool in enumerate(pools):
            _ext.kernels().paged_kv_append(kv[layer, 0].to(DEV), kv[layer, 1].to(DEV), pool.k, pool.v,
                                           bm.block_tables, r, p)
        at = 0
        for s, n in zip(seqs, counts):
            old = want.get(s)
            part = kv[:, :, at:at + n]
            want[s] = part if old is None else torch.cat([old, part], 2)
            at += n

    def check(seqs):
        q = torch.randn(len(seqs), 2, Hkv * G, hd, generator=g).to(torch.bfloat16)
        ql = [1 + i % 2 for i in range(len(seqs))]
        for layer, pool in enumerate(pools):
            bm.pool = pool
            out = PagedAttentionForward(PagedAttentionConfig(Hkv * G, hd)).forward_manager_shared(
                q.to(DEV), bm, seqs, torch.tensor(ql, dtype=torch.int32, device=DEV)).cpu().double()
            bm.pool = pools[0]
            for i, s in enumerate(seqs):
                n = want[s].shape[2]
                assert n == bm.seq_len(s)
                for t in range(2):
                    seen = n - ql[i] + t + 1
                    for h in range(Hkv * G):
                        if t >= ql[i]:
                            assert (out[i, t, h] == 0).all()
                            continue
                        k, v = want[s][layer, :, :seen, h // G].double()
                        p = torch.softmax(k @ q[i, t, h].double() * hd ** -0.5, 0)
                        tol = 2.0 ** -8 * (p @ v).abs() + (2.0 ** -8 + 2.0 ** -11) * (p @ v.abs())
                        assert ((out[i, t, h] - p @ v).abs() <= tol).all()
        _ext.check_status(0)

    bm.allocate_sequence(9)
    write([9], [150])
    bm.allocate_sequence(0)
    write([0], [75])
    for c in (1, 2, 3):
        bm.fork_sequence(0, c)
        want[c] = want[0].clone()
    assert bm.shared_prefix([0, 1, 2, 3])[1] == 64
    write([0, 1, 2, 3], [1, 2, 30, 5])
    check([0, 1, 2, 3])
    check([1, 9])
    for s, n in ((2, 70), (3, 10), (1, 76)):
        bm.truncate_sequence(s, n)
        want[s] = want[s][:, :, :n]
    bm.free_sequence(9)
    write([3, 0], [3, 20])
    check([0, 1, 2, 3])
    assert bm.compact()
    in_use = sum(1 for p in range(64) if pools[0].ref_count(p))
    assert max(p for s in range(4) for p in bm.sequence_page_chain(s)) < in_use
    check([0, 1, 2, 3])
    write([1, 2], [9, 1])
    check([2, 1])


def test_generator_forks_and_verifies():
    cfg = GPTConfig.tiny(vocab=512, seq=256)
    m = GPTModel(cfg, device=DEV, seed=1)
    gen = GPTGenerator(m, max_sequences=6, max_len=256, block_size=16)
    prompt = torch.randint(0, cfg.vocab_size, (100,), generator=torch.Generator().manual_seed(3))
    many = gen.generate([prompt], 12, num_samples=3)
    assert many[0] == many[1] == many[2]  # forks of one prompt take the same path
    want = many[0]
    ids = [gen.add_sequence(prompt)]
    ids += [gen.fork(ids[0]) for _ in range(2)]
    before = [gen.manager.seq_len(s) for s in ids]
    # drafts: the true continuation, a wrong second token, none
    new = gen.verify(ids, [want[1:5], [want[1], (want[2] + 1) % 512, want[3]], []])
    assert new[0][:4] == want[1:5] and len(new[0]) == 5
    assert new[1][0] == want[1] and len(new[1]) == 2 and new[1][1] == want[2]
    assert new[2] == [want[1]]
    assert [gen.manager.seq_len(s) for s in ids] == [before[0] + 5, before[1] + 2, before[2] + 1]
    # sampled verification with the model's own distribution as the draft's
    probs = torch.full((3, 2, cfg.vocab_size), 1.0 / cfg.vocab_size, device=DEV)
    out = gen.verify(ids, [[1, 2], [3], []], probs, temperature=1.0, uniforms=torch.rand(3, 3, device=DEV))
    assert all(1 <= len(o) <= 3 for o in out)
    for s in ids:
        gen.release(s)
    assert gen.pools[0].free_count() == gen.pools[0].total_count()
    _ext.check_status(0)
    assert not math.isnan(float(gen.pools[0].k.float().sum()))
