"""Shared pages of the KV cache on the host: reference counts, forks, copy-on-write, truncation, compaction, the
copies behind them and their refusals; draft verification against its definition; both used by the generator."""
import random

import pytest
import torch

from scirs_b200.inference import (BlockManager, BlockManagerConfig, GPTGenerator, InferenceError, KvPageConfig,
                                  KvPagePool, PagedAttentionConfig, PagedAttentionForward, copy_pages, verify_drafts)
from scirs_b200.models.gpt import GPTConfig, GPTModel

BS, HKV, HD = 4, 2, 8


def _manager(pages=24, layers=2, seqs=8, per_seq=8):
    pools = [KvPagePool(pages, KvPageConfig(block_size=BS, num_heads=HKV, head_dim=HD), "cpu") for _ in range(layers)]
    return pools, BlockManager(pools[0], BlockManagerConfig(seqs, per_seq), pools)


def _append(pools, bm, seq, values):
    """Token i of the sequence gets values[i] in every layer (plus the layer's number)."""
    rows, pos = bm.reserve([seq], [len(values)])
    for layer, pool in enumerate(pools):
        for p, x in zip(pos, values):
            page = bm.sequence_page_chain(seq)[p // BS]
            pool.k[page, p % BS] = x + layer
            pool.v[page, p % BS] = -(x + layer)


def _tokens(pools, bm, seq):
    out = []
    for layer, pool in enumerate(pools):
        chain = bm.sequence_page_chain(seq)
        k = [float(pool.k[chain[p // BS], p % BS, 0, 0]) - layer for p in range(bm.seq_len(seq))]
        v = [-float(pool.v[chain[p // BS], p % BS, 1, 3]) - layer for p in range(bm.seq_len(seq))]
        assert k == v
        out.append(k)
    assert all(o == out[0] for o in out)
    return out[0]


def test_fork_shares_until_written():
    pools, bm = _manager()
    bm.allocate_sequence(0)
    _append(pools, bm, 0, [1, 2, 3, 4, 5, 6])
    free = pools[0].free_count()
    bm.fork_sequence(0, 1)
    bm.fork_sequence(0, 2)
    assert pools[0].free_count() == free and bm.sequence_page_chain(1) == bm.sequence_page_chain(0)
    assert [pools[0].ref_count(p) for p in bm.sequence_page_chain(0)] == [3, 3]
    assert bm.shared_prefix([0, 1, 2]) == (bm.sequence_page_chain(0)[:1], BS)
    _append(pools, bm, 1, [7])
    _append(pools, bm, 0, [8])
    _append(pools, bm, 2, [9, 10, 11])  # the last holder writes in place, then grows
    assert _tokens(pools, bm, 0) == [1, 2, 3, 4, 5, 6, 8]
    assert _tokens(pools, bm, 1) == [1, 2, 3, 4, 5, 6, 7]
    assert _tokens(pools, bm, 2) == [1, 2, 3, 4, 5, 6, 9, 10, 11]
    assert pools[0].free_count() == free - 3
    for s in (0, 1, 2):
        bm.free_sequence(s)
    assert pools[0].free_count() == pools[0].total_count()


def test_truncate_gives_pages_back_and_respects_sharing():
    pools, bm = _manager()
    bm.allocate_sequence(0)
    _append(pools, bm, 0, list(range(10)))
    bm.fork_sequence(0, 1)
    bm.truncate_sequence(0, 2)
    assert len(bm.sequence_page_chain(0)) == 1 and bm.seq_len(0) == 2
    _append(pools, bm, 0, [50])  # slot 2 of a page that the fork still reads
    assert _tokens(pools, bm, 0) == [0, 1, 50]
    assert _tokens(pools, bm, 1) == list(range(10))
    bm.truncate_sequence(1, 0)
    assert len(bm.sequence_page_chain(1)) == 1
    with pytest.raises(InferenceError):
        bm.truncate_sequence(1, 1)


def test_fork_refusals_change_nothing():
    pools, bm = _manager(pages=3, seqs=2)
    bm.allocate_sequence(0)
    _append(pools, bm, 0, [1, 2, 3, 4, 5])
    with pytest.raises(InferenceError):
        bm.fork_sequence(5, 6)
    with pytest.raises(InferenceError):
        bm.fork_sequence(0, 0)
    bm.fork_sequence(0, 1)
    with pytest.raises(InferenceError):
        bm.fork_sequence(0, 2)  # no row left
    refs = [pools[0].ref_count(p) for p in range(3)]
    # one page is free: the copy of the shared page takes it, and nothing is left for a second one
    with pytest.raises(InferenceError):
        bm.reserve([0, 1], [1, 4])
    assert [pools[0].ref_count(p) for p in range(3)] == refs and bm.seq_len(0) == bm.seq_len(1) == 5
    _append(pools, bm, 1, [9])
    assert _tokens(pools, bm, 0) == [1, 2, 3, 4, 5] and _tokens(pools, bm, 1) == [1, 2, 3, 4, 5, 9]


def test_retained_pages_are_not_written_or_moved():
    pools, bm = _manager()
    bm.allocate_sequence(0)
    _append(pools, bm, 0, [1, 2])
    page = bm.sequence_page_chain(0)[0]
    pools[0].retain_page(page)  # a prefix cache, say
    _append(pools, bm, 0, [3])
    assert bm.sequence_page_chain(0)[0] != page and _tokens(pools, bm, 0) == [1, 2, 3]
    assert pools[0].ref_count(page) == 1
    pools[0].free_page(page)
    assert pools[0].ref_count(page) == 0
    with pytest.raises(InferenceError):
        pools[0].retain_page(page)


def test_random_operations_keep_every_sequence():
    rng = random.Random(0)
    pools, bm = _manager(pages=40, seqs=8, per_seq=8)
    want, nxt, value, moved = {}, 0, 0, 0
    for _ in range(600):
        op = rng.choice(["new", "append", "append", "fork", "fork", "truncate", "free", "compact", "append2"])
        live = list(want)
        try:
            if op == "new":
                bm.allocate_sequence(nxt)
                want[nxt], nxt = [], nxt + 1
            elif op == "fork" and live:
                s = rng.choice(live)
                bm.fork_sequence(s, nxt)
                want[nxt], nxt = list(want[s]), nxt + 1
            elif op in ("append", "append2") and live:
                some = rng.sample(live, min(len(live), 2 if op == "append2" else 1))
                counts = [rng.randint(0, 6) for _ in some]
                rows, pos = bm.reserve(some, counts)
                at = 0
                for s, n in zip(some, counts):
                    for p in pos[at:at + n]:
                        value += 1
                        for layer, pool in enumerate(pools):
                            page = bm.sequence_page_chain(s)[p // BS]
                            pool.k[page, p % BS] = value % 200 + layer
                            pool.v[page, p % BS] = -(value % 200 + layer)
                        want[s].append(value % 200)
                    at += n
            elif op == "truncate" and live:
                s = rng.choice(live)
                n = rng.randint(0, len(want[s]))
                bm.truncate_sequence(s, n)
                want[s] = want[s][:n]
            elif op == "free" and live:
                s = rng.choice(live)
                bm.free_sequence(s)
                del want[s]
            elif op == "compact":
                moved += len(bm.compact())
                used = {p for s in want for p in bm.sequence_page_chain(s)}
                assert used == set(range(len(used)))
        except InferenceError:
            pass
        held = {}
        for s in want:
            assert _tokens(pools, bm, s) == want[s]
            chain = bm.sequence_page_chain(s)
            assert bm._bt_host[bm.row_of(s), : len(chain)].tolist() == chain
            for p in chain:
                held[p] = held.get(p, 0) + 1
        assert all(pools[0].ref_count(p) == held.get(p, 0) for p in range(40))
        assert pools[0].free_count() == 40 - len(held) and len(set(pools[0]._free)) == len(pools[0]._free)
    assert moved > 0


def test_copy_pages_and_refusals():
    pools, _ = _manager(pages=6)
    for p in pools:
        p.k.normal_()
        p.v.normal_()
    before = [(p.k.clone(), p.v.clone()) for p in pools]
    copy_pages(pools, [0, 0, 1], torch.tensor([2, 3, 4], dtype=torch.int32), counts=[4, 2, 0])
    for p, (k, v) in zip(pools, before):
        for new, old in ((p.k, k), (p.v, v)):
            assert torch.equal(new[2], old[0]) and torch.equal(new[3, :2], old[0, :2])
            assert torch.equal(new[3, 2:], old[3, 2:]) and torch.equal(new[[0, 1, 4, 5]], old[[0, 1, 4, 5]])
    copy_pages(pools[0], [], [])
    state = [(p.k.clone(), p.v.clone()) for p in pools]
    for src, dst, counts in [([0], [6], None), ([-1], [1], None), ([0, 1], [2, 2], None), ([0, 1], [1, 2], None),
                             ([0], [1], [5]), ([0], [1], [-1]), ([0, 1], [2], None), ([0], [1], [1, 1])]:
        with pytest.raises(InferenceError):
            copy_pages(pools, src, dst, counts)
    with pytest.raises(InferenceError):
        copy_pages([], [0], [1])
    with pytest.raises(InferenceError):
        copy_pages(pools, torch.tensor([0]), [1])  # int64
    with pytest.raises(InferenceError):
        copy_pages([pools[0], KvPagePool(5, pools[0].config, "cpu")], [0], [1])
    assert all(torch.equal(p.k, k) and torch.equal(p.v, v) for p, (k, v) in zip(pools, state))


# ------------------------------------------------------------------------------------------------ verification
def test_verify_keeps_the_target_distribution():
    g = torch.Generator().manual_seed(5)
    N, V = 40000, 5
    p = torch.tensor([0.5, 0.2, 0.2, 0.1, 0.0])
    q = torch.tensor([0.1, 0.4, 0.2, 0.2, 0.1])
    x = torch.multinomial(q.expand(N, V), 1, generator=g)
    r = verify_drafts(p.expand(N, 2, V), q.expand(N, 1, V), x, torch.rand(N, 2, generator=g))
    emp = torch.bincount(r.tokens[:, 0], minlength=V) / N
    # 5 standard deviations of a frequency: 5 sqrt(p (1 - p) / N) <= 5 * 0.5 / 200
    assert (emp - p).abs().max() < 0.0125
    assert ((r.accepted == 1) == (r.tokens[:, 1] >= 0)).all()


def test_verify_edges():
    p = torch.tensor([[[0.0, 0.5, 0.5], [0.25, 0.25, 0.5]]])
    one = torch.tensor([[1]])

    def go(u0, u1, q=None, x=one, p=p, **kw):
        r = verify_drafts(p, q, x, torch.tensor([[u0, u1]]), **kw)
        return int(r.accepted[0]), r.tokens[0].tolist()

    # certain drafts: kept with probability p(x); the rest of p otherwise
    assert go(0.49, 0.0) == (1, [1, 0]) and go(0.5, 0.999) == (0, [2, -1])
    assert go(0.49, 0.25) == (1, [1, 1]) and go(0.49, 0.5) == (1, [1, 2])
    assert go(0.99, 0.0, acceptance_threshold=1.0) == (1, [1, 0])
    # equal distributions leave nothing: the row itself is drawn from, when the draft is refused all the same
    q = torch.tensor([[[0.0, 0.5, 0.5]]])
    assert go(0.3, 0.0, q) == (1, [1, 0])
    assert go(0.3, 0.0, q, x=torch.tensor([[0]])) == (0, [1, -1])  # q = 0 and p = 0
    assert go(0.3, 0.7, q, x=torch.tensor([[7]])) == (0, [2, -1])  # outside the vocabulary
    # no drafts, more lengths than drafts, padding behind the length
    assert go(0.0, 0.0, draft_lens=torch.tensor([0], dtype=torch.int32)) == (0, [1, -1])
    assert go(0.0, 0.0, draft_lens=torch.tensor([9], dtype=torch.int32)) == (1, [1, 0])
    r = verify_drafts(p[:, :1], None, torch.zeros(1, 0, dtype=torch.int64), torch.tensor([[0.6]]))
    assert r.accepted.tolist() == [0] and r.tokens.tolist() == [[2]]
    # values that are no weights
    bad = torch.tensor([[[float("nan"), float("inf"), 0.5], [0.0, -1.0, float("nan")]]])
    assert go(0.0, 0.99, x=torch.tensor([[0]]), p=bad) == (0, [2, -1])
    assert go(0.0, 0.5, x=torch.tensor([[2]]), p=bad) == (1, [2, -1])


def test_verify_refusals():
    p, q = torch.rand(2, 3, 7), torch.rand(2, 2, 7)
    x, u = torch.zeros(2, 2, dtype=torch.int64), torch.rand(2, 3)
    for bad in [(p[0], q, x, u), (p.double(), q.double(), x, u), (p, q[:, :1], x, u), (p, q.half(), x, u),
                (p, q, x.int(), u), (p, q, x[:, :1], u), (p, q, x, u.double()), (p, q, x, u[:, :2])]:
        with pytest.raises(ValueError):
            verify_drafts(*bad)
    for lens in (torch.tensor([1, 2]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError):
            verify_drafts(p, q, x, u, draft_lens=lens)


def test_attention_refusals():
    pool = KvPagePool(8, KvPageConfig(block_size=BS, num_heads=HKV, head_dim=HD), "cpu")
    att = PagedAttentionForward(PagedAttentionConfig(4, HD))
    bt, sl = torch.zeros(1, 3, dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    pages = torch.zeros(1, dtype=torch.int32)
    q = torch.randn(1, 4, HD)
    assert att.forward_shared_prefix(q, pool, bt, sl, pages, 4).shape == (1, 4, HD)
    for bad_q, n in [(torch.randn(1, 3, HD), 4), (torch.randn(1, 4, 16), 4), (q, 5), (q, -1)]:
        with pytest.raises(InferenceError):
            att.forward_shared_prefix(bad_q, pool, bt, sl, pages, n)
    with pytest.raises(InferenceError):
        PagedAttentionForward(PagedAttentionConfig(3, HD)).forward_shared_prefix(torch.randn(1, 3, HD), pool, bt, sl,
                                                                                pages, 4)


# ------------------------------------------------------------------------------------------------ the generator
def _generator(**kw):
    cfg = GPTConfig.tiny(vocab=128, seq=64)
    m = GPTModel(cfg, device="cpu", seed=1)
    return GPTGenerator(m, max_sequences=6, max_len=64, block_size=8, **kw)


def test_forked_samples_match_separate_prompts():
    prompt = torch.randint(0, 128, (13,), generator=torch.Generator().manual_seed(3))
    gen = _generator()
    one = gen.generate([prompt], 7)
    many = gen.generate([prompt, prompt[:5]], 7, num_samples=2)
    assert many[0] == many[1] == one[0] and many[2] == many[3] == gen.generate([prompt[:5]], 7)[0]
    assert gen.pools[0].free_count() == gen.pools[0].total_count()
    with pytest.raises(ValueError):
        gen.generate([prompt], 7, num_samples=0)


def test_verified_drafts_follow_greedy_generation():
    prompt = torch.randint(0, 128, (13,), generator=torch.Generator().manual_seed(3))
    gen = _generator()
    want = gen.generate([prompt], 12)[0]
    a = gen.add_sequence(prompt)
    b = gen.fork(a)
    rng = random.Random(2)
    got = {a: [gen.last_token[a]], b: [gen.last_token[b]]}
    while min(len(v) for v in got.values()) < 12:
        ids = [a, b]
        drafts = []
        for s in ids:
            true = want[len(got[s]):len(got[s]) + 3]
            drafts.append([t if rng.random() < 0.7 else (t + 1) % 128 for t in true][: rng.randint(0, 3)])
        for s, d, new in zip(ids, drafts, gen.verify(ids, drafts)):
            assert new[:-1] == d[: len(new) - 1] and len(new) >= 1
            got[s] += new
            assert gen.manager.seq_len(s) == 13 + len(got[s]) - 1
    assert got[a][:12] == got[b][:12] == want
    gen.release(a)
    gen.release(b)
    assert gen.pools[0].free_count() == gen.pools[0].total_count()


def test_verify_refuses_before_it_changes_anything():
    prompt = torch.randint(0, 128, (13,), generator=torch.Generator().manual_seed(3))
    gen = _generator()
    a = gen.add_sequence(prompt)
    V = 128
    for bad in [dict(drafts=[[1], [2]]), dict(drafts=[[V]]), dict(drafts=[[-1]]), dict(drafts=[[1] * 60]),
                dict(drafts=[[1]], draft_probs=torch.rand(1, 2, V)), dict(drafts=[[1]], uniforms=torch.rand(1, 1))]:
        with pytest.raises(InferenceError):
            gen.verify([a], **bad)
    with pytest.raises(InferenceError):
        gen.verify([a, a], [[1], [1]])
    assert gen.manager.seq_len(a) == 13
