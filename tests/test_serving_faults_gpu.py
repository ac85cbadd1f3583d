"""Serving operators on the GPU: calls that are refused, and places where a mistake would show only there."""
import pytest
import torch

from test_prefix_serving_gpu import Case

from scirs_b200 import _ext
from scirs_b200.inference import (GPTGenerator, InferenceError, KvPageConfig, KvPagePool, PagedAttentionConfig,
                                  PagedAttentionForward, copy_pages, verify_drafts)
from scirs_b200.models.gpt import GPTConfig, GPTModel
from scirs_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _generator(seqs=6, **kw):
    m = GPTModel(GPTConfig.tiny(vocab=512, seq=256), device=DEV, seed=1)
    return GPTGenerator(m, max_sequences=seqs, max_len=256, block_size=16, **kw)


def _prompt(n=100):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(3))


# ------------------------------------------------------------------------------------------------ refused calls
def test_refused_verification_leaves_the_sequences():
    gen = _generator()
    a = gen.add_sequence(_prompt())
    b = gen.fork(a)
    free = gen.pools[0].free_count()
    want = [gen.step([b])[0] for _ in range(3)]
    gen.release(b)
    probs = torch.full((1, 2, 512), 1 / 512)
    for bad in (dict(draft_probs=probs), dict(draft_probs=probs.double().to(DEV)), dict(uniforms=torch.rand(1, 3)),
                dict(uniforms=torch.rand(1, 3, device=DEV).double())):
        with pytest.raises(InferenceError):
            gen.verify([a], [[7, 9]], **bad)
        assert gen.manager.seq_len(a) == 100 and gen.pools[0].free_count() == free
    assert [gen.step([a])[0] for _ in range(3)] == want
    new = gen.verify([a], [[7, 9]], probs.to(DEV).to(torch.bfloat16), temperature=1.0)[0]
    assert gen.manager.seq_len(a) == 103 + len(new)
    _ext.check_status(0)


# ------------------------------------------------------------------------------------------------ samples
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_samples_of_logits_that_are_no_numbers_are_refused(value):
    """By the host: an assertion on the device would end all use of it."""
    gen = _generator()
    logits = torch.zeros(512, device=DEV)
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
    _ext.check_status(0)


def test_samples_begin_differently():
    gen = _generator()
    torch.manual_seed(0)
    # near to uniform over 512 tokens at temperature 50: six equal first tokens have odds of 512^-5
    assert len({o[0] for o in gen.generate([_prompt(), _prompt(20)], 3, temperature=50.0, num_samples=3)}) > 1
    assert gen.pools[0].free_count() == gen.pools[0].total_count()
    _ext.check_status(0)


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
    uniforms = torch.full((1, 2), 0.5, device=DEV)
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


# ------------------------------------------------------------------------------------------------ launches
def test_launches_are_counted_as_made():
    def launches(call):
        before = K.STATS.launches
        call()
        return K.STATS.launches - before

    def attend(B, rows, L):
        att = PagedAttentionForward(PagedAttentionConfig(rows, 64))
        pool = KvPagePool(L // 16 + 1, KvPageConfig(block_size=16, num_heads=1, head_dim=64), DEV)
        q = torch.zeros(B, rows, 64, dtype=torch.bfloat16, device=DEV)
        chain = torch.arange(L // 16 + 1, dtype=torch.int32, device=DEV)
        lens = torch.full((B,), L + 4, dtype=torch.int32, device=DEV)
        return lambda: att.forward_shared_prefix(q, pool, chain.expand(B, -1), lens, chain, L)

    assert launches(attend(4, 4, 512)) == 2  # 16 rows: the prefix goes with the tails
    assert launches(attend(5, 4, 512)) == 3  # 20 rows: tcgen05 takes it
    assert launches(attend(0, 4, 512)) == 0
    pools = [KvPagePool(2100, KvPageConfig(block_size=1, num_heads=1, head_dim=8), DEV) for _ in range(129)]
    assert launches(lambda: copy_pages(pools[:128], [0], [1])) == 1
    assert launches(lambda: copy_pages(pools, [0], [1])) == 2
    assert launches(lambda: copy_pages(pools[0], list(range(1025)), list(range(1025, 2050)))) == 2
    assert launches(lambda: copy_pages(pools, [], [])) == 0
    for B in (2, 0):
        p, x = torch.full((B, 2, 8), 0.125, device=DEV), torch.zeros(B, 1, dtype=torch.int64, device=DEV)
        assert launches(lambda: verify_drafts(p, p[:, :1], x, torch.zeros(B, 2, device=DEV))) == min(B, 1)
    _ext.check_status(0)


# ------------------------------------------------------------------------------------------------ bad pages
def _exact_without(c, lost):
    """(output, sum of p |v|) in 64 bits of a Case whose sequences do not see the keys of prefix pages `lost`; the
    tolerance is the one that Case.check derives."""
    o = torch.zeros(c.B, c.Q, c.Hkv * c.G, c.HD, dtype=torch.float64)
    a = torch.zeros_like(o)
    for b in range(c.B):
        m = int(c.lens[b])
        pos = torch.arange(m)
        page = c.tables[b].long()[pos // c.bs]
        kept = torch.ones(m, dtype=torch.bool)
        if m - c.Q + 1 >= c.L:
            for i in lost:
                kept &= (pos >= c.L) | (pos // c.bs != i)
        k, v = c.k[page, pos % c.bs].double(), c.v[page, pos % c.bs].double()
        for t in range(c.Q):
            on = kept & (pos < m - c.Q + t + 1)
            for h in range(c.Hkv * c.G):
                p = torch.softmax(k[on, h // c.G] @ c.q[b, t, h].double() * c.scale, 0)
                o[b, t, h], a[b, t, h] = p @ v[on, h // c.G], p @ v[on, h // c.G].abs()
    return o, a


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("B,L,HD,bs,lost", [
    (3, 90, 64, 16, [2]), (3, 90, 64, 8, [0, 11]), (3, 92, 128, 5, [7]), (3, 90, 40, 16, [5]),  # with the tails
    (20, 700, 64, 16, [7]), (20, 700, 128, 16, [0, 1, 9, 43]), (20, 700, 128, 128, [3]),  # tcgen05, copies by TMA
    (70, 640, 64, 64, [9]), (20, 641, 64, 5, [0, 60, 128]), (20, 650, 80, 16, [40])])  # and by cp.async; one block lost
def test_keys_of_bad_prefix_pages_are_left_out_on_every_path(B, L, HD, bs, lost, bad):
    c = Case([L + 3 + i % 7 for i in range(B)] + [L - 30], 2, 2, 2, HD, bs, L, seed=L + HD)
    o, a = _exact_without(c, lost)
    c.prefix_pages[lost] = bad
    out = c.run().cpu().double()
    with pytest.raises(RuntimeError, match="bounds"):
        _ext.check_status(0)
    err = (out - o).abs()
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * a + 1e-30
    assert torch.isfinite(out).all() and (err <= tol).all(), float((err / tol).max())


def test_a_block_of_bad_prefix_pages():
    """No key of the prefix's first two blocks is there, or none of it at all."""
    for lost in (list(range(16)), list(range(33)), list(range(8, 33))):
        c = Case([530] * 20, 1, 1, 2, 64, 16, 528, seed=2)
        o, a = _exact_without(c, lost)
        c.prefix_pages[lost] = -5
        out = c.run().cpu().double()
        with pytest.raises(RuntimeError, match="bounds"):
            _ext.check_status(0)
        assert ((out - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * a).all()


# ------------------------------------------------------------------------------------------------ inside the prefix
@pytest.mark.parametrize("lens,Q,Hkv,G,HD,bs,L,qlens", [
    # tcgen05 takes the prefix; one, some, most and all of the sequences end inside it
    pytest.param([2100] * 19 + [2040], 1, 2, 2, 128, 16, 2048, None, id="one_of_twenty"),
    pytest.param([2100, 3, 2060, 1999, 0, 1500] * 5, 2, 2, 2, 64, 16, 2048, [2, 2, 1, 2, 0, 1] * 5, id="a_third"),
    pytest.param([2047 - i for i in range(29)] + [2050], 1, 1, 8, 128, 16, 2048, None, id="all_but_one"),
    pytest.param([1600 + i for i in range(40)], 4, 1, 2, 64, 24, 1640, [4, 1, 2, 3] * 10, id="all"),
    pytest.param([2010, 2051, 2049, 1], 5, 2, 8, 128, 16, 2048, [5, 5, 1, 1], id="three_row_tiles_of_a_tail"),
    pytest.param([1800, 1700, 30] * 4, 2, 1, 2, 80, 16, 1750, None, id="head_dim_80"),
    pytest.param([1800, 1700, 30] * 4, 2, 2, 2, 64, 5, 1750, None, id="pages_of_five"),
    # the prefix goes with the tails (up to 16 rows)
    pytest.param([3000, 2980, 2, 2999], 1, 2, 4, 64, 16, 2990, None, id="items"),
    pytest.param([3000, 2980, 2, 2999], 2, 1, 2, 128, 5, 2990, [2, 2, 1, 2], id="items_cp_async"),
    # a warp a tail
    pytest.param([1300 if i % 9 else 1100 + i for i in range(100)], 1, 16, 1, 64, 16, 1250, None, id="warps"),
    pytest.param([1300 if i % 50 else 900 for i in range(100)], 2, 16, 1, 128, 16, 1250, [1 + i % 2 for i in range(100)],
                 id="warps_two_queries"),
    pytest.param([20000, 20040, 19000], 1, 8, 8, 128, 16, 20010, None, id="long"),
    # more keys than one item takes
    pytest.param([9100] * 11 + [9000], 1, 1, 2, 128, 16, 9040, None, id="long_one_of_twelve"),
    pytest.param([9100, 8300, 3, 9050, 0, 8999] * 2, 2, 1, 2, 64, 16, 9040, [2, 2, 1, 2, 0, 1] * 2, id="long_half"),
    pytest.param([9000 - 40 * i for i in range(12)], 1, 1, 2, 64, 16, 9040, None, id="long_all"),
    pytest.param([8400, 9050, 8999, 1], 5, 1, 8, 128, 16, 9040, [5, 5, 1, 1], id="long_three_row_tiles"),
    pytest.param([9100, 9000, 8500, 17], 2, 1, 3, 80, 16, 9040, None, id="long_head_dim_80"),
    pytest.param([9100, 9000, 8500, 17], 2, 1, 3, 64, 5, 9040, None, id="long_pages_of_five"),
    pytest.param([9100, 9000, 8500], 1, 2, 4, 64, 16, 9040, None, id="long_items"),
    pytest.param([9100, 9000, 8500], 2, 1, 2, 128, 5, 9040, [2, 2, 1], id="long_items_cp_async"),
    pytest.param([2300 if i % 9 else 2100 + i for i in range(100)], 1, 16, 1, 64, 16, 2250, None, id="long_warps"),
    pytest.param([2300 if i % 50 else 2200 for i in range(100)], 2, 16, 1, 128, 16, 2250, [1 + i % 2 for i in range(100)],
                 id="long_warps_two_queries"),
])
def test_sequences_that_end_inside_a_long_prefix(lens, Q, Hkv, G, HD, bs, L, qlens):
    c = Case(lens, Q, Hkv, G, HD, bs, L, qlens, seed=L + Q)
    first = c.run()
    c.check(first)
    pool = c.pool()
    assert all(torch.equal(c.run(pool=pool), first) for _ in range(3))


def test_a_sequence_that_ends_inside_the_prefix_in_a_graph():
    """A graph captured with lengths behind the prefix is replayed with some inside it, and the other way round."""
    c = Case([9100, 9060, 9070, 9060] * 5, 1, 1, 2, 64, 16, 9040, seed=6)
    pool = c.pool()
    c.k[:], c.v[:] = torch.nan_to_num(c.k), torch.nan_to_num(c.v)
    args = [t.to(DEV) for t in (c.q, c.tables, c.lens, c.prefix_pages)]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = c.att.forward_shared_prefix(args[0], pool, args[1], args[2], args[3], c.L)
    for lens in ([9100, 9030, 9070, 5] * 5, [9000] * 20, [9100, 9060, 9070, 9060] * 5):
        c.lens = torch.tensor(lens, dtype=torch.int32)
        args[2].copy_(c.lens)
        gr.replay()
        torch.cuda.synchronize()
        c.check(out)


def test_a_sequence_that_ends_inside_the_prefix_does_not_hold_up_the_batch():
    """Read by one item it took 14 times what the others take; in parts that spare items share, less than twice."""
    B, Hkv, G, HD, bs, L = 16, 8, 5, 128, 16, 65536
    n = L // bs
    pool = KvPagePool(2 * n + B, KvPageConfig(block_size=bs, num_heads=Hkv, head_dim=HD), DEV)
    pool.k.normal_()
    pool.v.normal_()
    front = torch.arange(n, dtype=torch.int32, device=DEV)
    tables = torch.cat([front.expand(B, -1), 2 * n + torch.arange(B, dtype=torch.int32, device=DEV)[:, None]], 1)
    tables[-1, :n] += n
    att = PagedAttentionForward(PagedAttentionConfig(Hkv * G, HD))
    q = torch.randn(B, Hkv * G, HD, device=DEV).to(torch.bfloat16)

    def time(last):
        lens = torch.tensor([L + 7] * (B - 1) + [last], dtype=torch.int32, device=DEV)
        took = []
        for i in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            att.forward_shared_prefix(q, pool, tables, lens, front, L)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b))
        return sorted(took)[3]

    behind, inside = time(L + 7), time(L - 9)
    _ext.check_status(0)
    assert inside < 5 * behind, (inside, behind)


# ------------------------------------------------------------------------------------------------ messages
def test_refusals_that_print_numbers():
    """Operands that do not match are an error with their sizes in it."""
    a, b = (torch.zeros(128, k, dtype=torch.bfloat16, device=DEV) for k in (64, 72))
    out = torch.zeros(128, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="64 vs 72"):
        K.gemm(a, b, out)
    with pytest.raises(RuntimeError, match="epilogue 99"):
        K.gemm(a, a, out, epi=99)
