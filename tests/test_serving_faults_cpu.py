"""Calls of the serving path that are refused or fail half way, samples at a temperature, logits and pages that are no
numbers: what is left behind, and what comes out."""
import pytest
import torch

from scirs_b200.inference import (BlockManager, BlockManagerConfig, GPTGenerator, InferenceError, KvPageConfig,
                                  KvPagePool, PagedAttentionConfig, PagedAttentionForward, SharedPrefixCache,
                                  verify_drafts)
from scirs_b200.models.gpt import GPTConfig, GPTModel

V = 128


def _generator(seqs=6):
    m = GPTModel(GPTConfig.tiny(vocab=V, seq=64), device="cpu", seed=1)
    return GPTGenerator(m, max_sequences=seqs, max_len=64, block_size=8)


def _prompt(n=13):
    return torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(3))


# ------------------------------------------------------------------------------------------------ refused calls
@pytest.mark.parametrize("bad", [
    dict(draft_probs=torch.full((2, 2, V), 1.0 / V, dtype=torch.float64)),
    dict(draft_probs=torch.ones(2, 2, V, dtype=torch.int64)),
    dict(draft_probs=torch.empty(2, 2, V, device="meta")),
    dict(uniforms=torch.rand(2, 3, dtype=torch.float64)),
    dict(uniforms=torch.rand(2, 3).to(torch.bfloat16)),
    dict(uniforms=torch.empty(2, 3, device="meta")),
])
def test_refused_verification_leaves_the_sequences(bad):
    gen = _generator()
    a = gen.add_sequence(_prompt())
    b = gen.fork(a)
    want = gen.step([a])[0], gen.step([a])[0]
    gen.release(a)
    free = gen.pools[0].free_count()
    c = gen.fork(b)
    with pytest.raises(InferenceError):
        gen.verify([b, c], [[7, 9], [3]], **bad)
    assert gen.manager.seq_len(b) == gen.manager.seq_len(c) == 13 and gen.pools[0].free_count() == free
    assert (gen.step([b])[0], gen.step([b])[0]) == want


def test_verification_that_fails_on_the_way_is_taken_back(monkeypatch):
    gen = _generator()
    a = gen.add_sequence(_prompt())
    pending, chain = gen.last_token[a], gen.manager.sequence_page_chain(a)
    want = gen.verify([a], [[7, 9, 11, 13]])
    gen.manager.truncate_sequence(a, 13)
    gen.last_token[a] = pending

    def fails(*args):
        raise RuntimeError("no memory")

    for call in (lambda: gen.verify([a], [[7, 9, 11, 13]]), lambda: gen.step([a])):
        with monkeypatch.context() as mp, pytest.raises(RuntimeError, match="no memory"):
            mp.setattr(gen, "_decode", fails)
            call()
        assert gen.manager.seq_len(a) == 13 and gen.last_token[a] == pending
        assert gen.manager.sequence_page_chain(a) == chain
    assert gen.verify([a], [[7, 9, 11, 13]]) == want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_draft_probabilities_of_sixteen_bits(dtype):
    """They count as the values that they hold."""
    q = torch.softmax(torch.randn(1, 3, V, generator=torch.Generator().manual_seed(1)), -1).to(dtype)
    u = torch.tensor([[0.3, 0.9, 0.2, 0.6]])
    out = []
    for probs in (q, q.float()):
        gen = _generator()
        a = gen.add_sequence(_prompt())
        out.append((gen.verify([a], [[5, 6, 7]], probs, temperature=1.0, uniforms=u), gen.manager.seq_len(a)))
    assert out[0] == out[1]


def test_verification_of_no_sequences():
    gen = _generator()
    assert gen.verify([], []) == []
    with pytest.raises(InferenceError):
        gen.verify([], [[1]])


# ------------------------------------------------------------------------------------------------ samples
@pytest.mark.parametrize("groups", [1, 8])
def test_first_tokens_of_samples_follow_the_distribution(groups):
    """N first tokens at a temperature, all of one prompt and in several calls."""
    N, T = 1600, 0.7
    gen = _generator(seqs=N // groups)
    gen._prefill = (lambda prefill: lambda p: (prefill(p)[0], logits))(gen._prefill)
    logits = torch.full((V,), float("-inf"))
    logits[[3, 50, 77, 127]] = torch.tensor([0.5, 0.25, 0.125, 0.125]).log() * T
    torch.manual_seed(7)
    first = []
    for _ in range(groups):
        first += [o[0] for o in gen.generate([_prompt(3)], 1, temperature=T, num_samples=N // groups)]
    assert len(first) == N
    emp = torch.bincount(torch.tensor(first), minlength=V) / N
    p = torch.softmax(logits / T, -1)
    # 5 standard deviations of a frequency: 5 sqrt(p (1 - p) / N) <= 5 * 0.5 / 40
    assert (emp - p).abs().max() < 0.0625 and emp[p == 0].sum() == 0


def test_samples_at_a_high_temperature_begin_differently():
    gen = _generator()
    torch.manual_seed(0)
    # the model's distribution at temperature 50 is near to uniform over 128: six equal first tokens have odds of 128^-5
    assert len({o[0] for o in gen.generate([_prompt()], 3, temperature=50.0, num_samples=6)}) > 1
    assert len({gen.generate([_prompt()], 2, temperature=50.0)[0][0] for _ in range(6)}) > 1
    assert gen.pools[0].free_count() == gen.pools[0].total_count()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_samples_of_logits_that_are_no_numbers_are_refused(value):
    """By the host: an assertion on the device would end all use of it."""
    gen = _generator()
    logits = torch.zeros(V)
    logits[slice(None) if value < 0 else 5] = value
    prefill, decode = gen._prefill, gen._decode
    gen._prefill = lambda p: (prefill(p)[0], logits)
    with pytest.raises(InferenceError, match="no token"):
        gen.generate([_prompt()], 2, temperature=1.0, num_samples=3)
    gen._prefill = prefill
    ids = [gen.add_sequence(_prompt()) for _ in range(2)]
    gen._decode = lambda *args: torch.stack([decode(*args)[0], logits])
    with pytest.raises(InferenceError, match="no token"):
        gen.step(ids, temperature=1.0)
    n = _prompt().numel()
    assert [gen.manager.seq_len(s) for s in ids] == [n, n]
    gen._decode = decode
    assert len(gen.step(ids, temperature=1.0)) == 2


# ------------------------------------------------------------------------------------------------ numbers that are none
@pytest.mark.parametrize("temperature,row", [(0.0, 0), (0.0, 1), (0.0, None), (1.0, 0), (1.0, None)])
def test_verification_of_logits_that_are_no_numbers(temperature, row):
    """Row 0 belongs to the pending token, row 1 to the draft (refused where it is not the model's choice)."""
    gen = _generator()
    a = gen.add_sequence(_prompt())
    size, pending, decode = gen.manager.seq_len(a), gen.last_token[a], gen._decode

    def nan(*args):
        lg = decode(*args)
        lg[slice(None) if row is None else row, 5] = float("nan")
        return lg

    best = gen.step([a])[0]
    gen.manager.truncate_sequence(a, size)
    gen.last_token[a] = pending
    gen._decode = nan
    uniforms = torch.full((1, 2), 0.5)
    if row == 1 and temperature == 0.0:  # a refused draft: its row is not looked at
        assert gen.verify([a], [[(best + 1) % 100]], temperature=temperature, uniforms=uniforms) == [[best]]
        gen.manager.truncate_sequence(a, size)
        gen.last_token[a] = pending
    draft = [best] if temperature == 0.0 else []
    with pytest.raises(InferenceError, match="no token"):
        gen.verify([a], [draft], temperature=temperature, uniforms=uniforms[:, : 1 + len(draft)])
    assert gen.manager.seq_len(a) == size and gen.last_token[a] == pending
    gen._decode = decode
    assert gen.step([a]) == [best]


# ------------------------------------------------------------------------------------------------ nothing left behind
def test_generation_that_finds_no_room_leaves_nothing_behind():
    gen = _generator(seqs=3)
    total = gen.pools[0].total_count()

    def empty():
        return (gen.manager.active_sequences() == 0 and gen.pools[0].free_count() == total and not gen.last_token
                and len(gen.manager._free_rows) == 3)

    with pytest.raises(InferenceError, match="too many"):
        gen.generate([_prompt()], 4, num_samples=4)
    assert empty()
    with pytest.raises(InferenceError, match="too many"):
        gen.generate([_prompt(), _prompt(5)], 4, temperature=1.0, num_samples=2)
    assert empty()
    # pages: two prompts fit, their third sequence finds none
    held = [gen.pools[0].alloc_page() for _ in range(total - 4)]
    total = 4
    with pytest.raises(InferenceError, match="exhausted"):
        gen.generate([_prompt(13), _prompt(13), _prompt(13)], 4)
    assert empty()
    with pytest.raises(InferenceError, match="exhausted"):  # the prompt's second page is not there
        gen.pools[0].retain_page(held[0])
        extra = [gen.pools[0].alloc_page() for _ in range(3)]
        gen.add_sequence(_prompt(13))
    total = 1
    assert empty()
    for p in extra:
        gen.pools[0].free_page(p)
    assert len(gen.generate([_prompt()], 4, num_samples=2)) == 2


# ------------------------------------------------------------------------------------------------ cached prefixes
def test_pages_of_a_prefix_cache_stay():
    pool = KvPagePool(8, KvPageConfig(block_size=4, num_heads=2, head_dim=8), "cpu")
    bm = BlockManager(pool, BlockManagerConfig(4, 8))
    cache = SharedPrefixCache(pool)

    def write(seq, n, value):
        kv = torch.full((n, 2, 8), value).to(torch.bfloat16)
        bm.append([seq], [n], kv, -kv)

    bm.allocate_sequence(0)
    write(0, 4, 1.0)
    bm.allocate_sequence(1)
    write(1, 8, 2.0)
    cache.insert(5, bm.sequence_page_chain(1))
    listed = list(cache.lookup(5))
    bm.fork_sequence(1, 2)
    write(2, 4, 3.0)
    bm.free_sequence(0)  # a hole in front of the listed pages
    moves = bm.compact()
    assert moves and cache.lookup(5) == listed == bm.sequence_page_chain(1)[:2] == bm.sequence_page_chain(2)[:2]
    bm.free_sequence(1)
    bm.free_sequence(2)
    assert [pool.ref_count(p) for p in listed] == [1, 1] and pool.free_count() == 6
    assert (pool.k[listed] == 2.0).all() and (pool.v[listed] == -2.0).all()
    # a refused entry changes nothing, another chain under the hash takes the place of the first, which is given back
    free = next(p for p in range(8) if pool.ref_count(p) == 0)
    with pytest.raises(InferenceError):
        cache.insert(5, [listed[0], free])
    assert cache.lookup(5) == listed and pool.ref_count(listed[0]) == 1
    cache.insert(5, listed[:1])
    assert [pool.ref_count(p) for p in listed] == [1, 0]
    assert cache.evict(5) == listed[:1] and cache.evict(5) is None and pool.free_count() == 8


# ------------------------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("n,vocab", [(1, 1 << 30), (1, (1 << 31) - 65), (1 << 30, 1)])
def test_verification_refuses_rows_of_more_than_thirty_bits(n, vocab):
    def like(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    with pytest.raises(ValueError, match="2\\^30"):
        verify_drafts(like(1, n + 1, vocab), like(1, n, vocab), like(1, n, dtype=torch.int64), like(1, n + 1))


# ------------------------------------------------------------------------------------------------ bad pages
@pytest.mark.parametrize("bad", [-1, 8, 10 ** 6])
def test_pages_outside_of_the_pool_are_refused(bad):
    pool = KvPagePool(8, KvPageConfig(block_size=4, num_heads=2, head_dim=8), "cpu")
    att = PagedAttentionForward(PagedAttentionConfig(2, 8))
    tables, lens = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32), torch.tensor([14], dtype=torch.int32)
    prefix, q = torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, 2, 8)
    assert att.forward_shared_prefix(q, pool, tables, lens, prefix, 8).shape == q.shape
    for t, i in ((tables[0], 3), (prefix, 1)):
        old = int(t[i])
        t[i] = bad
        with pytest.raises(InferenceError, match="outside"):
            att.forward_shared_prefix(q, pool, tables, lens, prefix, 8)
        t[i] = old
    tables[0, 3] = bad  # behind the sequence's end
    lens[0] = 12
    assert att.forward_shared_prefix(q, pool, tables, lens, prefix, 8).shape == q.shape


# ------------------------------------------------------------------------------------------------ the shared prefix
@pytest.mark.parametrize("queries", [1, 3, 20])
def test_the_managers_prefix_ends_in_front_of_the_queries(queries, monkeypatch):
    """Forks without tokens of their own, and one sequence alone, share full pages up to the newest token."""
    pool = KvPagePool(16, KvPageConfig(block_size=4, num_heads=2, head_dim=8), "cpu")
    bm = BlockManager(pool, BlockManagerConfig(4, 8))
    bm.allocate_sequence(0)
    kv = torch.randn(16, 2, 8, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    bm.append([0], [16], kv, kv.flip(0))
    bm.fork_sequence(0, 1)
    att = PagedAttentionForward(PagedAttentionConfig(4, 8))
    seen = []
    shared = PagedAttentionForward.forward_shared_prefix

    def spy(self, q, pool, tables, lens, pages, prefix_len, *rest):
        seen.append(prefix_len)
        return shared(self, q, pool, tables, lens, pages, prefix_len, *rest)

    monkeypatch.setattr(PagedAttentionForward, "forward_shared_prefix", spy)
    for seqs in ([0, 1], [0]):
        q = torch.randn(len(seqs), queries, 4, 8, generator=torch.Generator().manual_seed(1))
        out = att.forward_manager_shared(q, bm, seqs)
        assert seen.pop() == max(0, 16 - queries + 1)  # every query stands behind it
        none = torch.zeros(0, dtype=torch.int32)
        want = shared(att, q, pool, bm.block_tables[: len(seqs)][[bm.row_of(s) for s in seqs]],
                      bm.seq_lens[[bm.row_of(s) for s in seqs]], none, 0)
        assert torch.equal(out, want)


def test_sequences_that_share_nothing_are_not_walked(monkeypatch):
    """Growing them asks for no page's references, and nothing of their chains but the first pages is compared."""
    pool = KvPagePool(64, KvPageConfig(block_size=4, num_heads=1, head_dim=8), "cpu")
    bm = BlockManager(pool, BlockManagerConfig(4, 16))

    class Chain(list):
        def __getitem__(self, i):
            assert i == 0
            return list.__getitem__(self, i)

    for s in range(3):
        bm.allocate_sequence(s)
        bm.reserve([s], [14])
        bm._pages[s] = Chain(bm._pages[s])
    with monkeypatch.context() as mp:
        mp.setattr(pool, "ref_count", None)
        rows, pos = bm.reserve([0, 1, 2], [1, 5, 1])
        assert bm.shared_prefix([0, 1, 2]) == ([], 0)
    assert pos == [14, 14, 15, 16, 17, 18, 14] and bm.seq_len(1) == 19
    assert bm.shared_prefix([]) == ([], 0)
    bm._pages = {s: list(c) for s, c in bm._pages.items()}
    bm.fork_sequence(0, 3)
    assert bm.shared_prefix([0, 3]) == (bm.sequence_page_chain(0)[:3], 12)
    bm.reserve([3, 0], [1, 1])  # the last, partly filled page is copied
    assert bm.sequence_page_chain(0)[:3] == bm.sequence_page_chain(3)[:3]
    assert bm.sequence_page_chain(0)[3] != bm.sequence_page_chain(3)[3]
